// int4tc.cuh - the 4-bit linear layer for more than 16 rows of a 16-bit type, on tcgen05 (included by int4lin.cu).
//
// 128 outputs x up to 64 rows of x per CTA; a cluster of `split` CTAs divides the inputs. A stage is 128 inputs, two blocks
// of 64: warps 0-7 unpack 16 outputs each into the A operand (code - 8, exact in fp16 and bf16; 128 rows of 128 bytes,
// 128-byte swizzle), a thread of warp 9 has the tensor copies bring x's rows as the B operand, warp 8 issues the products.
// The sums of a group stay apart from the next one's: a unit (a stage, or 64 or 32 inputs with groups of those) has a buffer
// of TMEM columns, four in turn, that the warps 12-15 (an output per thread) read, multiply by the output's scale and add up
// in registers. Zero points enter as scale * (8 - zero) * the sum of x over the unit, which warps 9-11 take from the rows.
// A stage's fence stands before the next loads: behind them it waits for their data (x by cp.async and fences: 40 us for
// 48 rows, 4096 outputs of 14336 inputs; by tensor copies 27).
// Measured, bf16, groups of 128: 48 x 14336 -> 4096 27 us (29 MB of codes, 209 TFLOP/s; mma.sync 35.5), groups of 64 29, of
// 32 43; with zero points 58, 63 and 74; 64 x 14336 -> 16384 81 us (117 MB, 370 TFLOP/s; mma.sync 146); 4096 -> 4096 at 256 rows
// 30, at 1,024 112 us: the codes are unpacked again for every 64 rows. The roles wait for one another: the tensor pipe is
// active 13 % and the schedulers issue 35 % of the time; unpacking eight codes is seven logic and four floating-point
// instructions in eight warps, a wait that suspends resumes some hundred cycles late, and clusters, barriers and the sums at
// the end are 5 us of every call. With zero points three warps take the sums of
// every stage's rows beside (not profiled).
#pragma once

constexpr int kTcThreads = 512, kTcStages = 4, kTcBufs = 4, kTcCols = 64;
constexpr int kTcAhead = 3, kTcSums = 2 * kTcStages;       // stages from x's copy to its sums; stages whose sums are kept
static_assert(kTcAhead < kTcStages, "a stage's sums are taken before its refill waits for them");

struct TcSmem {
    uint8_t a[kTcStages][2][128 * 128];                    // two blocks of 64 inputs
    uint8_t b[kTcStages][2][64 * 128];
    float sx[kTcSums][4][64];                              // the sums of x over 32 inputs, by row
    uint64_t a_full[kTcStages], b_full[kTcStages], empty[kTcStages], sx_full[kTcSums], d_full[kTcBufs], d_empty[kTcBufs], done;
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(TcSmem::a) >= 64 * 128 * 4, "the sums fit the A stages");

template <int DT, bool ZERO, int US, int NC>               // 2^US units in a stage; NC: chunks of 32 rows
__global__ void __launch_bounds__(kTcThreads, 1) int4_tc(const __grid_constant__ Int4Args a,
                                                         const __grid_constant__ CUtensorMap tx, int split) {
    constexpr int ROWS = 32 * NC;
    constexpr uint32_t FMT = DT == F16 ? 0 : 1;            // operand types of the instruction descriptor
    constexpr uint32_t IDESC = idesc(kFmtF32, FMT, FMT, 0, 0, 128, ROWS);
    extern __shared__ uint8_t smem_raw[];
    TcSmem& sm = *reinterpret_cast<TcSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    volatile int* abort = &sm.abort;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = (int) (blockIdx.x % split), block = (int) (blockIdx.x / split), KT = (a.K + 63) / 64;
    const int per = ((KT + split - 1) / split + 1) / 2, stages = (KT + 1) / 2;
    const int kp0 = min(stages, part * per), n_it = min(stages, kp0 + per) - kp0;
    constexpr int UNITS = 1 << US, STEPS = 8 / UNITS;      // of a stage: 128, 64 or 32 inputs each
    const long long m0 = (long long) blockIdx.y * ROWS;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kTcStages; ++i) {
            mbar_init(sm.a_full + i, 8);
            mbar_init(sm.b_full + i, a.x_vec ? 1 : 96);
            mbar_init(sm.empty + i, 1);
        }
        for (int i = 0; i < kTcSums; ++i) mbar_init(sm.sx_full + i, 3);
        for (int i = 0; i < kTcBufs; ++i) {
            mbar_init(sm.d_full + i, 1);
            mbar_init(sm.d_empty + i, 4);
        }
        mbar_init(&sm.done, 1);
        sm.abort = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&sm.tmem, kTcBufs * kTcCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    static_assert(kTcBufs == kTcStages, "with a unit to a stage the unit's barrier frees the stage too");
    uint64_t* empty = US > 0 ? sm.empty : sm.d_full;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return warp_wait(bar, parity, a.wait_ns, abort); };
    bool ok = true;
    float acc[ROWS];
    if (warp < 8) {
        // ---------------- unpack: strip `warp` of the block ----------------
        const int g = lane >> 2, t = lane & 3;
        const int nt = min(block * 8 + warp, (a.N + 15) / 16 - 1);          // a strip past the last repeats it, unstored
        const uint4* src = a.tiles + (size_t) nt * KT * 32 + lane;
        uint4 w[kTcStages][2];
        auto fetch = [&](int it, int u) {                  // (past the last tile x is zeros)
            const int kt = 2 * (kp0 + it);
            w[u][0] = __ldcs(src + (size_t) kt * 32);
            w[u][1] = __ldcs(src + (size_t) min(kt + 1, KT - 1) * 32);
        };
#pragma unroll
        for (int u = 0; u < kTcStages; ++u)
            if (u < n_it) fetch(u, u);
        // the lane's two rows, g and g + 8 of the strip, have one swizzle (g); piece 4 h + t of both
        const uint32_t row = (uint32_t) (warp * 16 + g) * 128;
        for (int base = 0; base < n_it && ok; base += kTcStages) {
#pragma unroll
            for (int u = 0; u < kTcStages; ++u) {
                const int it = base + u;
                if (it >= n_it) break;
                uint4 f[2][2][2];
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const uint32_t words[4] = {w[u][v].x, w[u][v].y, w[u][v].z, w[u][v].w};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t lo[4], hi[4];
                        frag<DT>(words[2 * h], lo);
                        frag<DT>(words[2 * h + 1], hi);
                        f[v][h][0] = make_uint4(lo[0], lo[2], hi[0], hi[2]);
                        f[v][h][1] = make_uint4(lo[1], lo[3], hi[1], hi[3]);
                    }
                }
                if (it >= kTcStages && !wait(empty + u, ((it / kTcStages) & 1) ^ 1)) { ok = false; break; }
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint8_t* to = sm.a[u][v] + row + (uint32_t) (((4 * h + t) ^ g) << 4);
                        *reinterpret_cast<uint4*>(to) = f[v][h][0];
                        *reinterpret_cast<uint4*>(to + 8 * 128) = f[v][h][1];
                    }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(sm.a_full + u);
                if (it + kTcStages < n_it) fetch(it + kTcStages, u);       // (behind the fence, which would wait for it)
            }
        }
    } else if (warp == 8) {
        // ---------------- products ----------------
        const uint64_t da = sdesc(smem_u32(sm.a[0][0]), 16, 1024), db = sdesc(smem_u32(sm.b[0][0]), 16, 1024);
        uint32_t unit = 0;
        for (int it = 0; it < n_it && ok; ++it) {
            const int st = it % kTcStages;
            const uint32_t ph = (uint32_t) (it / kTcStages) & 1;
            ok = wait(sm.a_full + st, ph) && wait(sm.b_full + st, ph);
            const uint64_t sa = da + (uint32_t) (st * 2048), sb = db + (uint32_t) (st * 1024);   // (they count in 16 bytes)
#pragma unroll
            for (int u = 0; u < UNITS; ++u, ++unit) {
                const uint32_t buf = unit % kTcBufs;
                if (ok && unit >= kTcBufs) ok = wait(sm.d_empty + buf, ((unit / kTcBufs) & 1) ^ 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {          // 16 inputs of 2 bytes
                    const int kk = u * STEPS + i;
                    mma_ss_w<false>(tmem + buf * kTcCols, sa + (uint32_t) ((kk >> 2) * 1024 + (kk & 3) * 2),
                                    sb + (uint32_t) ((kk >> 2) * 512 + (kk & 3) * 2), IDESC, i > 0 ? 1u : 0u);
                }
                mma_commit_w(sm.d_full + buf);
            }
            if (US > 0 && ok) mma_commit_w(sm.empty + st);
        }
        mma_commit_w(&sm.done);                            // products in flight, also where a wait gave up
        warp_wait(&sm.done, 0, a.wait_ns, nullptr);
    } else if (warp < 12) {
        // ---------------- x: ROWS rows of 128 inputs; its sums, ROWS rows x 16 pieces of 8 inputs ----------------
        constexpr int X = (ROWS * 16 + 95) / 96, XS = 96 / 16;              // a thread's pieces; its rows are XS apart
        const int tid = (int) threadIdx.x - 9 * 32, c = tid & 15, r0 = tid >> 4;
        uint32_t to[X];                                    // (the swizzle is by the row)
#pragma unroll
        for (int j = 0; j < X; ++j) {
            const int r = r0 + j * XS;
            to[j] = smem_u32(sm.b[0][c >> 3]) + (uint32_t) (r * 128 + (((c & 7) ^ (r & 7)) << 4));
        }
        auto load = [&](int it) {
            uint64_t* bar = sm.b_full + it % kTcStages;
            if (a.x_vec) {                                 // past the rows and the inputs the copies bring zeros
                if (tid == 0) {
                    mbar_expect_tx(bar, 2 * ROWS * 128);
                    for (int v = 0; v < 2; ++v) tma_load_2d(sm.b[it % kTcStages][v], &tx, bar, (kp0 + it) * 128 + v * 64, (int) m0);
                }
                return;
            }
#pragma unroll
            for (int j = 0; j < X; ++j) {
                const int r = r0 + j * XS, k = (kp0 + it) * 128 + c * 8;
                if (r >= ROWS) continue;
                Raw<DT> x{};
                if (m0 + r < a.M && k < a.K) x = load_raw<DT>(a, static_cast<const char*>(a.x) + (size_t) (m0 + r) * a.K * 2, k, false);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to[j] + (uint32_t) (it % kTcStages) * (uint32_t) sizeof(sm.b[0])),
                             "r"(x.u[0].x), "r"(x.u[0].y), "r"(x.u[0].z), "r"(x.u[0].w) : "memory");
            }
            fence_proxy_async_smem();
            mbar_arrive(bar);
        };
        // Two warps have nothing to do where one thread's copies bring x and there are no sums to take: phases that nothing
        // holds for them could pass unseen, and a wait for one of them would then last to its limit.
        const int rounds = a.x_vec && !ZERO && warp != 9 ? 0 : n_it + (ZERO ? kTcAhead : 0);
        int issued = 0;
        for (int nx = 0; nx < rounds; ++nx) {
            if (nx < n_it) {
                // A stage is free once its products are complete and its sums have been taken. A thread that stores x takes
                // the sums of what it stored, earlier in this loop; one thread's copies write what all three warps read:
                // that one waits for the sums of the stage that leaves (sx_full cannot run ahead of this warp, which is
                // one of those that complete it). The other two follow by b_full alone, a phase of which waits for them.
                const int leaves = nx - kTcStages;
                if (leaves >= 0 && !(ZERO && a.x_vec && warp != 9)) {
                    ok = wait(empty + nx % kTcStages, ((nx / kTcStages) & 1) ^ 1);
                    if (ZERO && a.x_vec && ok) ok = wait(sm.sx_full + leaves % kTcSums, (leaves / kTcSums) & 1);
                    if (!ok) break;
                }
                load(nx);
                issued = nx + 1;
            }
            if (!ZERO || nx < kTcAhead) continue;
            const int it = nx - kTcAhead, st = it % kTcStages;
            if (!wait(sm.b_full + st, (it / kTcStages) & 1)) { ok = false; break; }
            if constexpr (ZERO) {                          // 4 lanes to 32 inputs of a row
#pragma unroll
                for (int j = 0; j < X; ++j) {
                    const int r = r0 + j * XS;
                    uint4 x = make_uint4(0u, 0u, 0u, 0u);
                    if (r < ROWS)
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(to[j] + (uint32_t) st * (uint32_t) sizeof(sm.b[0])) : "memory");
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                    float s = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) s += bits_value(w[e] & 0xffffu, DT) + bits_value(w[e] >> 16, DT);
                    s += __shfl_xor_sync(0xffffffffu, s, 1);
                    s += __shfl_xor_sync(0xffffffffu, s, 2);
                    if ((c & 3) == 0 && r < ROWS) sm.sx[it % kTcSums][c >> 2][r] = s;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sm.sx_full + it % kTcSums);
            }
        }
        if (a.x_vec && warp == 9)                          // copies in flight, of the warp that made them
            for (int it = max(0, issued - kTcStages); it < issued; ++it) warp_wait(sm.b_full + it % kTcStages, (it / kTcStages) & 1, a.wait_ns, nullptr);
    } else {
        // ---------------- sums: output n of this thread, every row ----------------
#pragma unroll
        for (int i = 0; i < ROWS; ++i) acc[i] = 0.0f;
        const int n = min(block * 128 + (warp & 3) * 32 + lane, a.N - 1);
        const uint32_t t_lane = tmem + ((uint32_t) ((warp & 3) * 32) << 16);
        auto group_at = [&](uint32_t unit) {               // the scale's place; past the inputs the last group's (x is zero)
            const int k = min(kp0 * 128 + (int) (unit << (7 - US)), a.K - 1);
            return (size_t) (k >> a.group_shift) * a.N + n;
        };
        const uint32_t units = (uint32_t) n_it << US;
        uint32_t s_next = 0, z_next = 0;
        if (units > 0) {
            s_next = ld_bits(a.scale, group_at(0), a.s_dt);
            if constexpr (ZERO) z_next = ld_bits(a.zero, group_at(0), a.s_dt);
        }
        for (uint32_t unit = 0; unit < units; ++unit) {
            const uint32_t buf = unit % kTcBufs;
            const float s = bits_value(s_next, a.s_dt), z = ZERO ? 8.0f - bits_value(z_next, a.s_dt) : 0.0f;
            if (unit + 1 < units) {
                s_next = ld_bits(a.scale, group_at(unit + 1), a.s_dt);
                if constexpr (ZERO) z_next = ld_bits(a.zero, group_at(unit + 1), a.s_dt);
            }
            if (!wait(sm.d_full + buf, (unit / kTcBufs) & 1)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint32_t d[32];
                tmem_ld32(t_lane + buf * kTcCols + c * 32, d);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[c * 32 + i] = fmaf(s, __uint_as_float(d[i]), acc[c * 32 + i]);
            }
            if constexpr (ZERO) {
                // A slot is written again 8 stages on, after the products 4 stages on, which wait for this unit's buffer.
                const int it = (int) (unit >> US), q0 = (int) (unit & (UNITS - 1)) * (4 / UNITS);
                const float sz = s * z;
                if (!wait(sm.sx_full + it % kTcSums, (it / kTcSums) & 1)) { ok = false; break; }
                for (int e = q0; e < q0 + 4 / UNITS; ++e) {
                    const float* sx = sm.sx[it % kTcSums][e];
#pragma unroll
                    for (int i = 0; i < ROWS; ++i) acc[i] = fmaf(sz, sx[i], acc[i]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sm.d_empty + buf);
        }
    }
    if (!ok && lane == 0) {
        atomicOr(a.err, kErrInt4);
        *abort = 1;
    }
    // every product has been read (or the wait for it has given up): the A stages take the sums. CTA p finishes the rows p,
    // p + split, ...; [source][row / split][output].
    tc_fence_before();
    if (split > 1) cluster_sync();
    else __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, kTcBufs * kTcCols);
    }
    const int rows = ROWS / split;
    float* sums = reinterpret_cast<float*>(sm.a);
    if (warp >= 12) {
        const uint32_t mine = smem_u32(sums);
        const int col = (warp & 3) * 32 + lane;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const uint32_t at = mine + (uint32_t) ((part * rows + r / split) * 128 + col) * 4;
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(at, (uint32_t) (r % split))), "f"(acc[r]) : "memory");
        }
    }
    if (split > 1) cluster_sync();
    else __syncthreads();
    for (int i = threadIdx.x; i < rows * 128; i += kTcThreads) {
        const int c = i % 128, r = i / 128, n = block * 128 + c;
        const long long m = m0 + r * split + part;
        if (n >= a.N || m >= a.M) continue;
        float y = 0.0f;
        for (int p = 0; p < split; ++p) y += sums[(p * rows + r) * 128 + c];
        if (!is_finite(y)) y = int4_exact(a, m, n);
        if (a.bias) y += a.bias[n];
        st_dt(a.out, (size_t) m * a.N + n, y, a.out_dt);
    }
}
