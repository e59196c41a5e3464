// attendtc.cu - attention over the 8-bit cache for many query rows (a prompt, or a part of one, behind what is cached of
// it), on tcgen05: two 128-row query tiles per CTA in the structure of attn_sage3 (attn3.cuh), causal, with grouped
// heads, and with the codes unpacked to fp16 on the way into shared memory.
//
// The rows of a kv head are its group's heads of every new token, row r = token * group + head, 256 to a CTA, one row per
// softmax thread. A key tile is two halves of 64 keys: two pages, or a page and the tail. Codes are exact in fp16, so
// Q.K^T is q . code and a half's scale enters with its softmax: arg = s * (rs ks) - m. Values keep their codes too: the
// page's scale vs enters as an exponent, a = 2^(arg + log2(vs / vref)) = p vs / vref, so P.V accumulates code * a over pages
// of different scales, and the row's sum takes a's sum over vs / vref. vref is the largest scale that the CTA meets; a
// page whose scale is under 2^-60 of it counts with that (its values, 127 codes at most, are lost beside vref's).
// The reference m of a row is moved when a half's largest a would pass 2^14, so that this becomes 2^6 (to 2^7): fp16 keeps its
// 11 bits of an a down to 2^-20 of the row's largest, and what it drops is 2^-31 of that. Where the second half moves it
// while the first one's weights stand in fp16, it moves by a whole number, and these are multiplied by an exact power of
// two: an a is rounded once, to fp16, which is 2^-11 of it beside the 2^-8 or 2^-11 of the output; the row's sum takes it
// unrounded. (Whole numbers for every move: 2.94e-4 off the definition instead of 2.76e-4, fp16's own rounding 2.07e-4, at
// 1,999 tokens behind 15,002, since a weight that sets the reference is 2^6 exactly otherwise.)
// q, and the tail's keys and values, are brought to fp16 by powers of two (per row; per head's tail): exact for 16-bit
// types except what is some 2^27 times smaller than the row's or the tail's largest.
//
// Warps: 1 and 3 issue the MMAs of the query tiles 0 and 1; 4-7 and 8-11 are the softmax of tiles 0 and 1; 12 and 13 unpack
// the two halves of the key tiles, 14 and 15 those of the value tiles (16 codes per lane and load; the next half's loads
// are under way while a half is unpacked). The 128 registers a thread that 512 threads start with are dealt out again: 168 to
// the softmax warps, 120 to the unpacking ones, 56 to warps 0-3 (128 x (56 + 2 x 168 + 120) = 65,536).
//
// Measured: 1,999 tokens behind 15,002 cached ones, 32 heads of 128 over 8, fp16: 654 us, 524 GFLOP at 802 TFLOP/s (0.48 of the
// measured dense rate). The tensor pipe is active 43 % of the time: 256 CTAs on 148 SMs are two rounds where 1.73 would do,
// and within a CTA the softmax (an exponential per score, 16 a clock and SM) takes about as long as the products.
#include <algorithm>
#include <atomic>

#include "attn3_softmax.cuh"
#include "kvcommon.cuh"

namespace h3 {
namespace {

template <int HD>
struct TcCfg {
    static constexpr int CB = 128 * 128;                     // column block: 128 rows x 64 features, 128-byte swizzle
    static constexpr int TILE = HD / 64 * CB;                // a 128-row tile of Q, K or V
    static constexpr int NK = HD == 64 ? 6 : 3, NV = HD == 64 ? 4 : 2;
    static constexpr int KSTEPS = HD / 16;
    static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + NK * TILE, OFF_RS = OFF_V + NV * TILE;
    static constexpr int OFF_BAR = OFF_RS + 256 * 4;
    static constexpr int NBAR = 2 * NK + 2 * NV + 10;
    static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;      // tmem address, abort, tail flags, reduction scratch
    static constexpr int SMEM = OFF_MISC + 320 + 1024;
    static constexpr int THREADS = 512, WARPS = THREADS / 32;
    static constexpr uint32_t IDESC_QK = idesc(kFmtF32, kFmtF16, kFmtF16, 0, 0, kTileM, 64);
    static constexpr uint32_t IDESC_PV = idesc(kFmtF32, kFmtF16, kFmtF16, 0, 1, kTileM, HD);
    static_assert(SMEM <= 232448, "shared memory budget of one sm_100 CTA");
};

// where 16-byte piece c (8 features) of row r lies in a tile of 128-byte rows, 64 features to a column block
__device__ __forceinline__ uint32_t swizzled(int cb_bytes, int r, int c) {
    return (uint32_t) ((c >> 3) * cb_bytes + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
// 16 codes -> 16 halves: code + 128 in the low bits of 1024's mantissa, less 1152
__device__ __forceinline__ void codes16(const uint4 u, uint4& lo, uint4& hi) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t h[8];
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = w[i] ^ 0x80808080u;
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off), hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        h[2 * i] = *reinterpret_cast<const uint32_t*>(&ha);
        h[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hb);
    }
    lo = make_uint4(h[0], h[1], h[2], h[3]);
    hi = make_uint4(h[4], h[5], h[6], h[7]);
}
// the exponent e that brings top into [2^13, 2^14) when divided by 2^e, and 2^-e in two normal factors
__device__ __forceinline__ int exponent_of(float top) { return top > 0.0f ? ilogbf(top) - 13 : 0; }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }   // |e| <= 126
// 2^d of a whole d <= 0, 0 below 2^-126 (the conversion saturates: also for -infinity)
__device__ __forceinline__ float pow2_down(float d) { return __int_as_float(max(0, 127 + __float2int_rz(d)) << 23); }
__device__ __forceinline__ uint4 halves8(const float (&x)[8], float m1, float m2) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = pack_half2(x[2 * i] * m1 * m2, x[2 * i + 1] * m1 * m2);
    return make_uint4(h[0], h[1], h[2], h[3]);
}

template <int DT, int HD>
__global__ void __launch_bounds__(TcCfg<HD>::THREADS, 1) attend_tc(const __grid_constant__ AttendArgs a) {
    using C = TcCfg<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t* k_empty = k_full + C::NK;
    uint64_t* v_full = k_empty + C::NK;
    uint64_t* v_empty = v_full + C::NV;
    uint64_t* hi_full = v_empty + C::NV;   // [tile]: S_hi_t(j) complete
    uint64_t* lo_full = hi_full + 2;       // [tile]: S_lo_t(j) complete (and every earlier MMA); a last phase after the last P.V
    uint64_t* hi_free = lo_full + 2;       // [tile], one arrival per softmax warp: S_hi_t(j) read into registers
    uint64_t* p_full = hi_free + 2;        // [tile], one arrival per softmax warp: P_t(j) in TMEM, O_t rescaled
    uint64_t* mma_done = p_full + 2;       // [tile]: every MMA of that tile's issuer complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::OFF_MISC);
    volatile int* abort = reinterpret_cast<volatile int*>(sm + C::OFF_MISC + 4);
    float* scratch = reinterpret_cast<float*>(sm + C::OFF_MISC + 16);      // [4][16]
    float* rs = reinterpret_cast<float*>(sm + C::OFF_RS);

    const KvArgs& kv = a.kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.Hq / kv.heads, nz = a.plan.nz;
    const int h = (int) (blockIdx.x % kv.heads), z = blockIdx.y;
    let_next_launch();
    // which sequence's tile this is: the tiles of all sequences one after the other, a prefix sum over the sequences
    int* const found = reinterpret_cast<int*>(sm + C::OFF_MISC + 8);
    {
        int* const sums = reinterpret_cast<int*>(scratch);
        const int flat = (int) (blockIdx.x / kv.heads);
        if (threadIdx.x == 0) found[0] = -1;
        int before = 0;
        for (int b0 = 0; b0 < kv.seqs; b0 += C::THREADS) {
            const int i = b0 + (int) threadIdx.x;
            int n = 0;
            if (i < kv.seqs) {
                const Seq q = load_seq(kv, a.starts, a.T, i);
                if (q.ok) n = (q.n * group + 255) / 256;
                else atomicOr(kv.err, kErrLen);
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            __syncthreads();
            if (lane == 31) sums[warp] = upto;
            __syncthreads();
            int all = 0, mine = before;
            for (int w = 0; w < C::WARPS; ++w) {
                if (w < warp) mine += sums[w];
                all += sums[w];
            }
            const int from = mine + upto - n;
            if (flat >= from && flat < from + n) {
                found[0] = i;
                found[1] = n - 1 - (flat - from);          // a sequence's last tile, which sees the most keys, first
            }
            before += all;
        }
        __syncthreads();
    }
    const int b = found[0], tile = found[1];
    if (b < 0) return;                                     // fewer tiles than the grid has room for
    const Seq s = load_seq(kv, a.starts, a.T, b);
    const int R = s.n * group, full = s.L / kPage;
    const int* table = kv.table + (size_t) b * kv.width;
    const size_t tbase = ((size_t) b * kv.heads + h) * kPage * HD;         // this head's tail, in elements
    const int r0 = tile * 256, nrow = min(R - r0, 256);
    const int last_pos = s.L - s.n + (r0 + nrow - 1) / group;
    const Pieces pc = pieces(s.L, last_pos, nz);
    if (z >= max(pc.nu, 1)) return;
    const int p0 = min(z * pc.cz, pc.np), pages = min(pc.np, p0 + pc.cz) - p0;
    const bool tail = z == pc.tail_at;
    const int nh = pages + (tail ? 1 : 0), n_kv = (nh + 1) / 2, nkey = s.L - full * kPage;
    if (n_kv == 0) {                                       // rows that see nothing
        for (int i = threadIdx.x; i < nrow * HD; i += C::THREADS) {
            const int r = i / HD;
            const size_t gr = (size_t) (s.s0 + (r0 + r) / group) * a.Hq + h * group + (r0 + r) % group;
            st1<DT>(a.out, gr * HD + i % HD, 0.0f);
            if (a.lse && i % HD == 0) a.lse[gr] = INFINITY;
        }
        return;
    }
    auto page_of = [&](int i) -> int {                     // half i's page, or -1: the tail, nothing, or a bad page
        if (i >= pages) return -1;
        const int id = table[p0 + i];
        return page_ok(kv, id) ? id : -1;
    };
    auto slot_of = [&](int i) { return (i < pages ? p0 + i : full) * kPage; };

    // ---- all threads: barriers, TMEM, the largest value scale, the tail's exponents, Q
    if (threadIdx.x == 0) {
        // a K or V stage is full once both of its unpacking warps have written it, free once both MMA warps have committed
        // their last use of it
        for (int i = 0; i < C::NK; ++i) { mbar_init(k_full + i, 2); mbar_init(k_empty + i, 2); }
        for (int i = 0; i < C::NV; ++i) { mbar_init(v_full + i, 2); mbar_init(v_empty + i, 2); }
        for (int t = 0; t < 2; ++t) {
            mbar_init(hi_full + t, 1);
            mbar_init(lo_full + t, 1);
            mbar_init(hi_free + t, 4);
            mbar_init(p_full + t, 4);
            mbar_init(mma_done + t, 1);
        }
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    float vmax = 0.0f, tk = 0.0f, tv = 0.0f;
    bool odd = false;                                  // an infinity or a NaN among the tail's values
    for (int i = threadIdx.x; i < pages; i += C::THREADS) {
        const int id = table[p0 + i];
        if (page_ok(kv, id)) vmax = fmaxf(vmax, kv.vs[(size_t) id * kv.heads + h]);
        else atomicOr(kv.err, kErrPage);
    }
    if (tail)
        for (int i = threadIdx.x; i < nkey * HD / 8; i += C::THREADS) {
            float x[8];
            floats8(raw8<DT>(kv.tk, tbase + i * 8, true), x);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (finite(x[u])) tk = fmaxf(tk, fabsf(x[u]));
            floats8(raw8<DT>(kv.tv, tbase + i * 8, true), x);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (finite(x[u])) tv = fmaxf(tv, fabsf(x[u]));
                else odd = true;
            }
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
        tk = fmaxf(tk, __shfl_xor_sync(0xffffffffu, tk, o));
        tv = fmaxf(tv, __shfl_xor_sync(0xffffffffu, tv, o));
    }
    odd = __any_sync(0xffffffffu, odd);
    if (lane == 0) {
        scratch[warp] = vmax;
        scratch[1 * C::WARPS + warp] = tk;
        scratch[2 * C::WARPS + warp] = tv;
        scratch[3 * C::WARPS + warp] = odd ? 1.0f : 0.0f;
    }
    // Q as fp16 times a power of two per row: HD / 16 lanes to a row, 16 features each
    constexpr int LPR = HD / 16;
    for (int r = threadIdx.x / LPR; r < 256; r += C::THREADS / LPR) {
        const int i = threadIdx.x % LPR;
        float x[2][8] = {};
        if (r < nrow) {
            const size_t at = (size_t) (s.s0 + (r0 + r) / group) * a.qs + (size_t) (h * group + (r0 + r) % group) * HD + i * 16;
            ld8<DT>(a.q, at, a.q_vec, x[0]);
            ld8<DT>(a.q, at + 8, a.q_vec, x[1]);
        }
        float top = 0.0f;
#pragma unroll
        for (int u = 0; u < 16; ++u)
            if (finite(x[u / 8][u % 8])) top = fmaxf(top, fabsf(x[u / 8][u % 8]));
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(__activemask(), top, o));
        const int e = exponent_of(top), e1 = e / 2, e2 = e - e1;
        uint8_t* q = sm + (r >> 7) * C::TILE;
        *reinterpret_cast<uint4*>(q + swizzled(C::CB, r & 127, 2 * i)) = halves8(x[0], pow2(-e1), pow2(-e2));
        *reinterpret_cast<uint4*>(q + swizzled(C::CB, r & 127, 2 * i + 1)) = halves8(x[1], pow2(-e1), pow2(-e2));
        if (i == 0) rs[r] = a.scale_log2 * pow2(e1) * pow2(e2);
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    vmax = tk = tv = 0.0f;
    odd = false;
#pragma unroll
    for (int i = 0; i < C::WARPS; ++i) {
        vmax = fmaxf(vmax, scratch[i]);
        tk = fmaxf(tk, scratch[1 * C::WARPS + i]);
        tv = fmaxf(tv, scratch[2 * C::WARPS + i]);
        odd |= scratch[3 * C::WARPS + i] != 0.0f;
    }
    const int ek = exponent_of(tk), ev = exponent_of(tv);
    const float tks = pow2(ek / 2) * pow2(ek - ek / 2), tvs = pow2(ev / 2) * pow2(ev - ev / 2);
    float vref = tail ? fmaxf(vmax, tvs) : vmax;
    if (!(vref > 0.0f)) vref = 1.0f;
    auto fail = [&](int code) {
        atomicOr(a.wait_err, code);
        *abort = 1;
    };
    auto ring = [&](uint32_t j, int n) { return (int) (j % n); };
    auto phase = [&](uint32_t j, int n) { return (j / n) & 1; };

    if (warp >= 12) {
        // ---------------- codes -> fp16 tiles: warps 12, 13 K, 14, 15 V; each a half of every tile ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        const bool is_k = warp < 14;
        const int sub = warp & 1, ns = is_k ? C::NK : C::NV;
        uint64_t* fullb = is_k ? k_full : v_full;
        uint64_t* empty = is_k ? k_empty : v_empty;
        const int8_t* codes = is_k ? kv.k : kv.v;
        const void* tl = is_k ? kv.tk : kv.tv;
        const int e = is_k ? ek : ev;
        constexpr int RPL = 32 / LPR, N = 64 / RPL;        // key rows of a warp's load, loads of a half
        // where this lane's first 8 features of load i go: the row of a load changes the swizzle by its bit 2 only
        const int r0l = lane / LPR, c0 = lane % LPR * 2;
        const uint32_t at0 = (uint32_t) ((c0 >> 3) * C::CB + (sub * 64 + r0l) * 128 + (((c0 & 7) ^ (r0l & 7)) << 4));
        auto place = [&](int i) { return (at0 ^ (uint32_t) (((i * RPL) & 4) << 4)) + (uint32_t) (i * RPL * 128); };
        auto source = [&](int id) {
            return reinterpret_cast<const uint4*>(codes + ((size_t) max(id, 0) * kv.heads + h) * kPage * HD) + lane;
        };
        bool ok = true;
        // a half's codes; each load of the next half is made where the code that it replaces has been unpacked, a whole
        // tile's time before it is needed. The page ids run one half further ahead.
        uint4 buf[N];
        int id = page_of(sub), next = page_of(sub + 2);
        if (id >= 0) {
            const uint4* src = source(id);
#pragma unroll
            for (int i = 0; i < N; ++i) buf[i] = src[i * 32];
        }
        for (int j = 0; j < n_kv; ++j) {
            const int st = j % ns, half = 2 * j + sub, after = page_of(half + 4);
            uint8_t* to = sm + (is_k ? C::OFF_K : C::OFF_V) + st * C::TILE;
            if (j >= ns && !warp_wait(empty + st, ((j / ns) & 1) ^ 1, a.wait_ns, abort)) { ok = false; break; }
            const uint4* src = source(next);
            if (id >= 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    uint4 lo, hi;
                    codes16(buf[i], lo, hi);
                    *reinterpret_cast<uint4*>(to + place(i)) = lo;
                    *reinterpret_cast<uint4*>(to + (place(i) ^ 16u)) = hi;
                    if (next >= 0) buf[i] = src[i * 32];
                }
            } else {                                       // the tail, or nothing: no codes follow the tail
                for (int i = 0; i < N; ++i) {
                    const int r = i * RPL + r0l;
                    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
                    if (tail && half == pages && r < nkey) {
                        float x[2][8];
                        floats8(raw8<DT>(tl, tbase + (size_t) r * HD + c0 * 8, true), x[0]);
                        floats8(raw8<DT>(tl, tbase + (size_t) r * HD + c0 * 8 + 8, true), x[1]);
                        if (!is_k)                         // 0 * infinity would reach rows that do not see it: added at the end
#pragma unroll
                            for (int v = 0; v < 16; ++v)
                                if (!finite(x[v / 8][v % 8])) x[v / 8][v % 8] = 0.0f;
                        lo = halves8(x[0], pow2(-(e / 2)), pow2(-(e - e / 2)));
                        hi = halves8(x[1], pow2(-(e / 2)), pow2(-(e - e / 2)));
                    }
                    *reinterpret_cast<uint4*>(to + place(i)) = lo;
                    *reinterpret_cast<uint4*>(to + (place(i) ^ 16u)) = hi;
                }
                if (next >= 0)                             // after a page that is out of the pool
#pragma unroll
                    for (int i = 0; i < N; ++i) buf[i] = src[i * 32];
            }
            id = next;
            next = after;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(fullb + st);
        }
        if (!ok && lane == 0) fail(kErrCache);
    } else if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
      if (warp & 1) {
        // ---------------- MMA issuers: warp 1 for query tile 0, warp 3 for tile 1 ----------------
        const int t = warp == 1 ? 0 : 1;
        auto qk = [&](uint32_t j, int half) {
            tc_fence_after();
            const uint32_t q_base = smem_u32(sm + t * C::TILE);
            const uint32_t k_base = smem_u32(sm + C::OFF_K + ring(j, C::NK) * C::TILE + half * 64 * 128);
#pragma unroll
            for (int kk = 0; kk < C::KSTEPS; ++kk) {
                const uint32_t off = (uint32_t) ((kk / 4) * C::CB + (kk % 4) * 32);
                mma_ss_w<false>(tmem + t * kTileN + half * 64, sdesc(q_base + off, 16, 1024), sdesc(k_base + off, 16, 1024),
                                C::IDESC_QK, kk > 0 ? 1u : 0u);
            }
        };
        auto pv = [&](uint32_t j, bool start) {
            tc_fence_after();
            const uint32_t v_base = smem_u32(sm + C::OFF_V + ring(j, C::NV) * C::TILE);
#pragma unroll
            for (int kk = 0; kk < kTileN / 16; ++kk)
                mma_ts_f16_w(tmem + 2 * kTileN + t * HD, tmem + t * kTileN + kk * 8,
                             sdesc(v_base + (uint32_t) (kk * 16 * 128), C::CB, 1024), C::IDESC_PV,
                             (!start || kk > 0) ? 1u : 0u);
        };
        auto wait_k = [&](uint32_t j) { return warp_wait(k_full + ring(j, C::NK), phase(j, C::NK), a.wait_ns, abort); };
        auto wait_v = [&](uint32_t j) { return warp_wait(v_full + ring(j, C::NV), phase(j, C::NV), a.wait_ns, abort); };
        bool ok = wait_k(0);
        if (ok) {
            qk(0, 1);
            mma_commit_w(hi_full + t);
            qk(0, 0);
            mma_commit_w(k_empty);
            mma_commit_w(lo_full + t);
        }
        for (int i = 0; i < n_kv && ok; ++i) {
            const uint32_t j = (uint32_t) i;
            const bool more = i + 1 < n_kv;
            if (!wait_v(j) || (more && !wait_k(j + 1))) { ok = false; break; }
            if (more) {
                if (!warp_wait(hi_free + t, j & 1, a.wait_ns, abort)) { ok = false; break; }
                qk(j + 1, 1);
                mma_commit_w(hi_full + t);
            }
            if (!warp_wait(p_full + t, j & 1, a.wait_ns, abort)) { ok = false; break; }
            pv(j, i == 0);
            mma_commit_w(v_empty + ring(j, C::NV));
            if (more) {
                qk(j + 1, 0);
                mma_commit_w(k_empty + ring(j + 1, C::NK));
            }
            mma_commit_w(lo_full + t);
        }
        if (!ok && lane == 0) fail(kErrCache);
        mma_commit_w(mma_done + t);
        mbar_wait(mma_done + t, 0, a.wait_ns, nullptr);
        __syncwarp();
      }
    } else {
        // ---------------- softmax + epilogue: warps 4-7 tile 0, warps 8-11 tile 1 ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        const int t = (warp - 4) >> 2, wq = warp & 3;
        const int row = wq * 32 + lane, r = t * 128 + row;
        const uint32_t t_lane = tmem + ((uint32_t) (wq * 32) << 16);
        const uint32_t colS = (uint32_t) (t * kTileN), colO = (uint32_t) (2 * kTileN + t * HD);
        const bool live = r < nrow;
        const int tok = (r0 + r) / group, hq = h * group + (r0 + r) % group;
        const int pos = live ? s.L - s.n + tok : -1;
        const float cq = rs[r];
        float m_run = -INFINITY, l_run = 0.0f;
        bool ok = true;
        // a half's scales and the keys that this row sees of it; loaded one tile ahead
        struct Half {
            float ks, vs;
            int valid;
        };
        auto half_of = [&](int i) {
            Half x;
            const int id = page_of(i);
            const bool is_tail = tail && i == pages;
            x.valid = id >= 0 || is_tail ? pos + 1 - slot_of(i) : 0;
            x.ks = id >= 0 ? kv.ks[(size_t) id * kv.heads + h] : tks;
            x.vs = id >= 0 ? kv.vs[(size_t) id * kv.heads + h] : tvs;
            return x;
        };
        Half lo = half_of(0), hi = half_of(1);
        const uint32_t bar_to1 = 1 + 2 * wq, bar_to0 = 2 + 2 * wq;
        auto take_turn = [&](bool start) {
            if (t == 1) bar_sync(bar_to1, 64);
            else if (!start) bar_sync(bar_to0, 64);
        };
        auto give_turn = [&] { bar_arrive(t == 0 ? bar_to1 : bar_to0, 64); };
        int turns = 0;
        for (int i = 0; i < n_kv; ++i) {
            const uint32_t j = (uint32_t) i;
            // c > 0 always, so -inf keys stay -inf through the FFMA
            const float c_lo = fmaxf(cq * lo.ks, 1e-30f), c_hi = fmaxf(cq * hi.ks, 1e-30f);
            const float w_lo = fmaxf(lo.vs / vref, 8.7e-19f), w_hi = fmaxf(hi.vs / vref, 8.7e-19f);
            const float g_lo = __log2f(w_lo), g_hi = __log2f(w_hi);
            const int valid_lo = lo.valid, valid_hi = hi.valid;
            lo = half_of(2 * i + 2);
            hi = half_of(2 * i + 3);
            const float m_prev = m_run;

            // ---- keys 64-127: read, free the columns for the next tile, max, exps (P_hi stays in registers)
            ok = warp_wait(hi_full + t, j & 1, a.wait_ns, abort);
            if (!ok) break;
            tc_fence_after();
            uint32_t x[2][32];
            tmem_ld32(t_lane + colS + 64, x[0]);
            tmem_ld32(t_lane + colS + 96, x[1]);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(hi_free + t);
            const float sm_hi = sage3_bias_max<false>(x, valid_hi) * c_hi + g_hi;
            if (sm_hi > m_run + 14.0f) m_run = sm_hi - 6.0f;
            const float m_hi = m_run;
            uint32_t p_hi[32];
            take_turn(turns == 0);
            float sum_hi = sage3_exp_half(x, c_hi, m_run == -INFINITY ? 0.0f : g_hi - m_run, p_hi);
            give_turn();
            ++turns;

            // ---- keys 0-63: read (after P(j-1).V_{j-1}), max, and where the max moves, scale P_hi down
            ok = warp_wait(lo_full + t, j & 1, a.wait_ns, abort);
            if (!ok) break;
            tc_fence_after();
            tmem_ld32(t_lane + colS, x[0]);
            tmem_ld32(t_lane + colS + 32, x[1]);
            tmem_wait_ld();
            const float sm_lo = sage3_bias_max<false>(x, valid_lo) * c_lo + g_lo;
            float up = 0.0f;                           // how far the reference moves while P_hi stands in fp16: a whole number
            if (sm_lo > m_run + 14.0f) {
                up = m_hi == -INFINITY ? INFINITY : floorf(sm_lo - m_hi) - 6.0f;
                m_run = m_hi == -INFINITY ? sm_lo - 6.0f : m_hi + up;
            }
            if (__any_sync(0xffffffffu, up != 0.0f)) {
                const float f = pow2_down(-up);
                const __half2 f2 = __float2half2_rn(f);
                sum_hi *= f;
#pragma unroll
                for (int u = 0; u < 32; ++u) {
                    __half2 v = *reinterpret_cast<__half2*>(&p_hi[u]);
                    v = __hmul2(v, f2);
                    p_hi[u] = *reinterpret_cast<uint32_t*>(&v);
                }
            }
            uint32_t p_lo[32];
            take_turn(false);
            tmem_st16(t_lane + colS + 32, *reinterpret_cast<const uint32_t(*)[16]>(&p_hi[0]));
            tmem_st16(t_lane + colS + 48, *reinterpret_cast<const uint32_t(*)[16]>(&p_hi[16]));
            const float sum_lo = sage3_exp_half(x, c_lo, m_run == -INFINITY ? 0.0f : g_lo - m_run, p_lo);
            give_turn();
            ++turns;
            tmem_st16(t_lane + colS, *reinterpret_cast<const uint32_t(*)[16]>(&p_lo[0]));
            tmem_st16(t_lane + colS + 16, *reinterpret_cast<const uint32_t(*)[16]>(&p_lo[16]));
            const bool grow = m_run != m_prev;
            const float alpha = grow ? (m_prev == -INFINITY ? 0.0f : ex2(m_prev - m_run)) : 1.0f;
            l_run = fmaf(l_run, alpha, sum_hi / w_hi + sum_lo / w_lo);
            if (__any_sync(0xffffffffu, grow && i > 0)) {
                const float al = i > 0 ? alpha : 1.0f;
#pragma unroll
                for (int c4 = 0; c4 < HD / 32; ++c4) {
                    uint32_t o[32];
                    tmem_ld32(t_lane + colO + c4 * 32, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int u = 0; u < 32; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * al);
                    tmem_st32(t_lane + colO + c4 * 32, o);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + t);
        }
        // the turns this warp has left after a failure, without work
        if (!ok && lane == 0) fail(kErrCache);
        for (; turns < 2 * n_kv; ++turns) {
            take_turn(turns == 0);
            give_turn();
        }
        // tile 1's last hand-back is taken here, so that no named barrier is left half arrived
        if (t == 0) bar_sync(bar_to0, 64);
        // the final P_t.V: the MMA warp commits lo_full once more after the last one
        if (ok) ok = warp_wait(lo_full + t, n_kv & 1, a.wait_ns, abort);
        if (!ok) {
            if (lane == 0) fail(kErrCache);
        } else {
            tc_fence_after();
            const size_t gr = (size_t) (s.s0 + tok) * a.Hq + hq;
            const bool split = pc.nu > 1;
            const float f = split ? vref : l_run == 0.0f ? 0.0f : vref / l_run;
            const bool added = tail && odd;
#pragma unroll
            for (int c4 = 0; c4 < HD / 32; ++c4) {
                uint32_t o[32];
                __syncwarp();                          // the loads are the whole warp's; what follows is each row's own
                tmem_ld32(t_lane + colO + c4 * 32, o);
                tmem_wait_ld();
                if (live) {
                    float y[32];
#pragma unroll
                    for (int u = 0; u < 32; ++u) y[u] = l_run == 0.0f ? 0.0f : __uint_as_float(o[u]) * f;
                    if (added) {                           // the tail's infinities and NaN, where this row sees them
                        for (int k = 0; k < min(nkey, pos + 1 - full * kPage); ++k)
#pragma unroll
                            for (int u = 0; u < 32; ++u) {
                                const float v = ld1<DT>(kv.tv, tbase + (size_t) k * HD + c4 * 32 + u);
                                if (!finite(v)) y[u] += v;
                            }
                    }
                    if (split) {
                        float4* to = reinterpret_cast<float4*>(a.part + (gr * nz + z) * HD + c4 * 32);
#pragma unroll
                        for (int u = 0; u < 8; ++u) to[u] = make_float4(y[4 * u], y[4 * u + 1], y[4 * u + 2], y[4 * u + 3]);
                    } else if (a.out_vec) {
                        uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(a.out) + (gr * HD + c4 * 32) * 2);
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if constexpr (DT == F16) w[e] = pack_half2(y[8 * u + 2 * e], y[8 * u + 2 * e + 1]);
                                else {
                                    const __nv_bfloat162 v = __floats2bfloat162_rn(y[8 * u + 2 * e], y[8 * u + 2 * e + 1]);
                                    w[e] = *reinterpret_cast<const uint32_t*>(&v);
                                }
                            }
                            to[u] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int u = 0; u < 32; ++u) st1<DT>(a.out, gr * HD + c4 * 32 + u, y[u]);
                    }
                }
            }
            if (live && split) {
                float* ml = a.part + (size_t) a.plan.entries * HD + (gr * nz + z) * 2;
                ml[0] = m_run;
                ml[1] = l_run;
            } else if (live && a.lse) {
                a.lse[gr] = l_run == 0.0f ? INFINITY : m_run + log2f(l_run);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <int DT, int HD>
cudaError_t launch(const AttendArgs& a, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = allow_smem(ready, attend_tc<DT, HD>, TcCfg<HD>::SMEM);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned) (a.kv.heads * a.plan.grid), (unsigned) a.plan.nz);
    attend_tc<DT, HD><<<grid, TcCfg<HD>::THREADS, TcCfg<HD>::SMEM, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attend_tc(const AttendArgs& a, cudaStream_t st) {
    if (a.kv.dt == F16) return a.kv.dim == 64 ? launch<F16, 64>(a, st) : launch<F16, 128>(a, st);
    return a.kv.dim == 64 ? launch<BF16, 64>(a, st) : launch<BF16, 128>(a, st);
}

}  // namespace h3
