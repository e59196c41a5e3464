// kvcache.cuh - the argument block and the launchers of the 8-bit key/value cache (kvcache.cu): h3s_kv_append,
// h3s_attention_cached, h3s_kv_evict. The layout and the meaning of every field stand at h3s_kv_cache in
// include/h3cuda.h.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace h3 {

constexpr int kPage = 64;              // tokens of a page: the Sage quantiser's block, with one scale per head
constexpr int kErrPage = 1;            // index errors (the second word of a context's error words): a page id
constexpr int kErrCache = 64;          // a wait of the attention over the cache gave up (the first error word)
constexpr int kErrLen = 2;             //   lens or starts out of range

struct KvArgs {
    int8_t* k;                         // [pages, heads, 64, dim]
    int8_t* v;
    float* ks;                         // [pages, heads]
    float* vs;
    void* tk;                          // [seqs, heads, 64, dim] in dt: the tokens that do not fill a page yet
    void* tv;
    float* w;                          // [pages, heads, 64] or NULL: the attention weight that each token received
    float* tw;                         // [seqs, heads, 64]
    int* table;                        // [seqs, width] page ids
    int* lens;                         // [seqs]
    long long pages;
    int seqs, width, heads, dim, dt;
    int* err;                          // index errors
};

// How a call's queries and keys are divided (the same on the host and in every kernel of one call).
struct AttendPlan {
    int rows;                          // query rows of a tile: 8 or 16, or 256 on tcgen05
    // 8 or 16 rows: a CTA for each piece that there can be of all (sequence, tile, head) units, units + room of them, whatever
    // the hints; those without a piece return at once. The pieces have about as many pages as make `room` of them (0: every
    // unit is one piece). 256: `grid` tiles (of all sequences) x heads x nz splits of the keys, one to a CTA.
    int grid, room, nz;
    bool joined;                       // partial results may be left, which attend_join brings together
    long long entries;                 // of partial rows
};
AttendPlan attend_plan(int n_sm, int dt, int64_t seqs, int64_t heads, int64_t group, int64_t T, int64_t max_new, int64_t max_len);

struct AttendArgs {
    KvArgs kv;
    const void* q;
    long long T, qs;                   // query rows, their stride (elements)
    int Hq;
    int group_shift, head_shift;       // log2 of Hq / heads and of heads, or -1: a division is 100 cycles of a short step's start
    const int* starts;                 // [seqs + 1]
    void* out;                         // [T, Hq * dim]
    float* part;                       // [entries, dim] accumulators, [entries, 2] (max, sum), and an int2 per sequence: its
                                       // first piece and the pieces of one of its units
    float* lse;                        // [T * Hq] or NULL: log2 of the softmax's sum, for the weights
    AttendPlan plan;
    long long max_new;
    float scale_log2;                  // log2(e) / sqrt(dim)
    int q_vec, out_vec;                // 16-byte loads of q's rows and stores of out's allowed
    int* wait_err;                     // device error word of waits that gave up
    unsigned long long wait_ns;        // limit of every wait
};
cudaError_t launch_attend(const AttendArgs& a, int n_sm, cudaStream_t st);

cudaError_t launch_attend_tc(const AttendArgs& a, cudaStream_t st);   // attendtc.cu

cudaError_t launch_kv_append(const KvArgs& kv, const void* k, const void* v, long long T, long long stride, const int* starts,
                             long long max_new, bool vec, cudaStream_t st);
cudaError_t launch_kv_evict(const KvArgs& kv, int* spare, int budget, int sinks, int recent, int* kept, cudaStream_t st);

}  // namespace h3
