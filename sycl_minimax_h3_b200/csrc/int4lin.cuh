// int4lin.cuh - the argument block and the launchers of the 4-bit linear layer (int4lin.cu): h3s_int4_linear,
// h3s_int4_pack.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace h3 {

// W[n, k] = scale[k / group, n] * (code[n, k] - zero[k / group, n]), zero = 8 where there is none.
struct Int4Args {
    const void* x;                     // [M, K] in x_dt
    const uint4* tiles;                // [ceil(N / 16), ceil(K / 64), 32 lanes]: see int4lin.cu
    const void* scale;                 // [groups, N] in s_dt
    const void* zero;                  // the same, or NULL
    const float* bias;                 // [N] or NULL
    void* out;                         // [M, N] in out_dt
    long long M;
    int N, K, group_shift;             // groups of 2^group_shift inputs: 5 to 7, or 30 (one scale for each output)
    int x_dt, s_dt, out_dt;
    int x_vec;                         // 16-byte loads of x's rows allowed
    int* err;                          // device error word of waits that gave up
    unsigned long long wait_ns;        // limit of every wait
};
cudaError_t launch_int4_linear(const Int4Args& a, int n_sm, cudaStream_t st);
cudaError_t launch_int4_pack(const uint8_t* codes, long long N, long long K, void* tiles, int n_sm, cudaStream_t st);

}  // namespace h3
