/* h3cuda.h - the C ABI of libh3cuda.so: the denoiser self-attention path of MiniMax H3 on NVIDIA B200 (sm_100a).
 *
 * A drop-in for the attention subset of the reference's kernels/h3sycl.h (maxfridbe/sycl_minimax_h3): the same names,
 * signatures, element-type codes and error conventions, with SYCL queues replaced by CUDA streams and USM by cudaMalloc.
 * Each declaration cites the reference declaration it replaces (file:line inside the reference project).
 *
 * Every data pointer is a device pointer of the context's GPU. Kernels are asynchronous: a call returns once its work
 * is queued on the context's stream, and the stream is in order, so a later call sees an earlier call's result;
 * h3s_read and h3s_wait are the points that wait. Functions returning int give 0, or -1 with the reason in
 * h3s_last_error() (per thread). Functions returning a pointer give NULL on failure, same.
 *
 * Environment (read when a context is made; same meanings as the reference's, kernels/h3sycl.cpp:216-235):
 *   H3S_ATTN=onednn (or =sdpa)  never use the int8 Sage path
 *   H3S_SAGE_MIN_S             sequences at least this long use Sage (default 8192)
 *   H3S_MEM_FRACTION           allocation cap as a fraction of the card (default 0.94)
 *   H3S_PROFILE                wait after every attention phase and report its time on stderr
 *   H3S_POISON                 fill new buffers with 0xff bytes (NaN) to expose reads of unwritten memory
 *   H3S_WAIT_MS                limit of every wait inside a kernel (default 2000); past it the kernel stops and
 *                              h3s_wait reports the failure
 */
#ifndef H3CUDA_H
#define H3CUDA_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types of floating-point tensors (kernels/h3sycl.h:21) */
enum { H3S_F32 = 0, H3S_F16 = 1, H3S_BF16 = 2 };

/* kernels/h3sycl.h:23 */
const char* h3s_last_error(void);

/* ---- context ---------------------------------------------------------------------------------------------------- */

/* A context on the first GPU with its own stream (kernels/h3sycl.h:28). */
void* h3s_open(void);
/* The GPUs CUDA sees; name, memory size and PCI address "0000:0b:00.0" of one (kernels/h3sycl.h:31-32). */
int h3s_gpu_count(void);
int h3s_gpu_info(int index, char* name, int name_len, uint64_t* mem_bytes, char* pci, int pci_len);
/* A context on GPU `index` with its own stream (kernels/h3sycl.h:33). */
void* h3s_open_gpu(int index);
/* A context around an existing stream: `stream` points to a cudaStream_t (PyTorch: the handle of
 * torch.cuda.current_stream()), which is copied; the current device is the context's GPU (kernels/h3sycl.h:36). */
void* h3s_create(void* stream);
/* Waits for the stream, frees the scratch buffers and everything still allocated with h3s_alloc (kernels/h3sycl.h:38). */
void h3s_destroy(void* ctx);
/* kernels/h3sycl.h:40 */
const char* h3s_device_name(void* ctx);

/* ---- device memory (kernels/h3sycl.h:47-53) --------------------------------------------------------------------- */

/* Allocations are counted, and one that would pass the cap (0.94 of the card; H3S_MEM_FRACTION overrides) is refused
 * with an error. The attention's own scratch buffers count against the same cap. */
void* h3s_alloc(void* ctx, uint64_t bytes);
void h3s_free(void* ctx, void* p); /* waits for the stream first */
uint64_t h3s_mem_used(void* ctx);
uint64_t h3s_mem_cap(void* ctx);
/* What the whole card has free right now, every process counted. */
uint64_t h3s_mem_free(void* ctx);

/* ---- copies (kernels/h3sycl.h:56-61) ---------------------------------------------------------------------------- */

/* Host <-> device; both wait for the copy (and for the work queued before it). Thread-safe. */
int h3s_write(void* ctx, void* dst, const void* src_host, uint64_t bytes);
int h3s_read(void* ctx, void* dst_host, const void* src, uint64_t bytes);
/* Device to device, queued like a kernel. */
int h3s_copy(void* ctx, void* dst, const void* src, uint64_t bytes);
/* Waits until everything queued has run; reports an asynchronous error (a CUDA error, or a kernel wait that gave up). */
int h3s_wait(void* ctx);

/* ---- pinned host memory and uploads beside the kernels (kernels/h3sycl.h:65-71) --------------------------------- */

void* h3s_alloc_host(void* ctx, uint64_t bytes);
void h3s_free_host(void* ctx, void* p); /* waits for the uploads first */
/* Pinned host -> device on the context's copy stream; the kernels do not wait for it: call h3s_upload_wait before
 * using dst. src must come from h3s_alloc_host, dst must be device memory; anything else is refused. */
int h3s_upload(void* ctx, void* dst, const void* src_pinned, uint64_t bytes);
int h3s_upload_wait(void* ctx);

/* ---- attention (kernels/h3sycl.h:185-197) ----------------------------------------------------------------------- */

/* out = softmax(q . k^T / sqrt(D)) . v, per head. q, k, v: S token rows of H heads x D features, row s at element
 * s * stride (stride >= H * D; 3 * H * D when they sit inside the qkv linear's output), in type dt; out [S, H * D] in
 * out_dt, rounded through half. S >= H3S_SAGE_MIN_S (8192): SageAttention v1 (int8 q, k with per-64-row scales after
 * k's channel mean is taken out; libh3sage.so beside this library) for D = 64 or 128, as the reference's plugin
 * (kernels/sage.cpp:33); every other call, and every D from 1 to 128, fp16 SDPA. D > 128 returns -1: a narrowing of
 * the reference, whose fused path takes any D (kernels/h3sycl.cpp:1464-1573); the engine's heads are 128 (denoiser)
 * and 64 (VAE). S, H or D <= 0: nothing to do, returns 0. No score table is ever written: memory stays O(S * H * D).
 * (kernels/h3sycl.h:190-191) */
int h3s_attention(void* ctx, const void* q, const void* k, const void* v, int dt, int64_t S, int64_t H, int64_t D,
                  int64_t stride, void* out, int out_dt);
/* B independent sequences of S tokens in one call: sequence b's rows start at row b * S of q, k, v and of out
 * [B * S, H * D]. Below the Sage threshold all sequences go in one launch; Sage takes them one at a time.
 * (kernels/h3sycl.h:196-197) */
int h3s_attention_batch(void* ctx, const void* q, const void* k, const void* v, int dt, int64_t B, int64_t S, int64_t H,
                        int64_t D, int64_t stride, void* out, int out_dt);

/* ---- the step before the attention (kernels/h3sycl.h:165-174) --------------------------------------------------- */

/* Per-head RMS norm, then the rotary position rotation, in place: what the denoiser runs on q and k right before
 * h3s_attention (engine/h3-core/src/dit.rs:347-348). x holds M token rows of H heads x D features, row m at element
 * m * stride (stride >= H * D), in type x_dt. Each head's features are normalised, s = sum of x*x in feature order,
 * inv = rsqrt(s / D + eps) (rounded once), x*inv*weight[i] (weight float [D]); then the pairs (i, rot_dim/2 + i),
 * i < rot_dim/2, are rotated by the token's angle, a' = a*cos - b*sin, b' = b*cos + a*sin, with (cos, sin) from cs
 * float [M, rot_dim/2, 2]. Features from rot_dim on are only normalised. rot_dim must be even, at most D, and leave an
 * even remainder, else -1. M, H or D <= 0: nothing to do, returns 0. Queued on the context's stream; no scratch. */
int h3s_rms_rope(void* ctx, void* x, int x_dt, int64_t M, int64_t H, int64_t D, int64_t stride, const float* weight,
                 float eps, const float* cs, int rot_dim);

/* ---- the block's linear layers (kernels/h3sycl.h:74-85) ----------------------------------------------------------- */

/* A linear layer with int8 weights and activations quantised on the fly (the int8_convrot checkpoints' layers: qkv,
 * out_proj, fc1, fc2 of every denoiser block, engine/h3-core/src/ops.rs:25-80):
 *
 *   x_rot = x . H           per group of `group` features, H the normalised Hadamard matrix h4 (x) h4 (x) ...
 *   s_r   = max(max|x_rot[r]| / 127, 1e-30)                  per row
 *   q     = clamp(rint(x_rot / s_r), -128, 127)              int8
 *   acc   = q . W^T                                          int32, on the tensor cores
 *   out   = acc * (s_r * wscale) + bias    (n_wscale = 1)    or   (acc * s_r) * wscale[n] + bias   (n_wscale = N)
 *
 * x [M, K] in x_dt; w int8 [N, K]; wscale float32 [n_wscale]; bias float32 [N] or NULL; out [M, N] in out_dt.
 * group = 0: no rotation; else a power of 2 up to 256 dividing K (as the reference accepts; 4^n is what checkpoints
 * use), else -1 "unsupported ConvRot group size". n_wscale must be 1 or N. M, K or N <= 0: nothing to do, returns 0.
 * Queued on the context's stream; the int8 copy of x is context scratch (grow-only, at most 1 GiB: longer inputs
 * run in row chunks). */
int h3s_int8_linear(void* ctx, const void* x, int x_dt, int64_t M, int64_t K, const int8_t* w, int64_t N,
                    const float* wscale, int64_t n_wscale, const float* bias, void* out, int out_dt, int group);

/* ---- the text encoder's attention (kernels/h3sycl.h:105-108) ---------------------------------------------------- */

/* Causal attention with grouped heads, for short sequences (the text encoder, engine/h3-core/src/te.rs:340-346): Hq
 * query heads share Hkv key/value heads (query head h reads key/value head h / (Hq / Hkv)). q rows of stride qs, k and
 * v rows of stride kvs (elements), type dt; out [L, Hq * D] in dt. Query i attends to keys 0..i with scores
 * q.k / sqrt(D), and every weight stays fp32 (nothing is rounded to half between the loads and the store).
 * D <= 256 and Hq a multiple of Hkv, else -1; L <= 0: nothing to do, returns 0. Queued on the context's stream. */
int h3s_attention_causal(void* ctx, const void* q, const void* k, const void* v, int dt, int64_t L, int64_t Hq,
                         int64_t Hkv, int64_t D, int64_t qs, int64_t kvs, void* out);

/* ---- additions without a counterpart in the reference ----------------------------------------------------------- */

/* The Ulysses exchange over peer memory, for one process per GPU on one node (NVLink/NVSwitch): a sequence of S
 * tokens sharded by tokens over P ranks (s = S/P rows each) is re-sharded by heads (h = H/P each) for the attention
 * and back, each rank storing straight into the other ranks' buffers.
 * h3s_ipc_handle: the 64-byte CUDA IPC handle of a buffer from h3s_alloc (its base pointer). h3s_ipc_open: another
 * process's buffer from its handle (NULL on failure); h3s_ipc_close undoes it. */
int h3s_ipc_handle(void* ctx, const void* ptr, void* handle);
void* h3s_ipc_open(void* ctx, const void* handle);
int h3s_ipc_close(void* ctx, void* ptr);
/* Forward: this rank's token rows of a qkv buffer, shard [s, 3*H*D] (q | k | v, es-byte elements: 2 or 4), into every
 * rank p's head-sharded buffer dst[p] = [P*s, 3*h*D]: heads p*h .. p*h+h-1 of each part, at rows rank*s .. rank*s+s-1.
 * Inverse: this rank's output out_heads [P*s, h*D] into every rank p's token rows dst[p] = [s, H*D] at columns
 * rank*h*D ... dst[rank] is this rank's own buffer, the others opened with h3s_ipc_open; P <= 8, H a multiple of P.
 * Queued on the context's stream; the ranks must meet (a collective on the same streams) before they overwrite what
 * another rank still reads and before they read what they received. */
int h3s_ulysses_push_qkv(void* ctx, const void* shard, int64_t s, int64_t H, int64_t D, int es, int P, int rank,
                         void* const* dst);
int h3s_ulysses_push_out(void* ctx, const void* out_heads, int64_t s, int64_t H, int64_t D, int es, int P, int rank,
                         void* const* dst);
/* h3s_attention of this rank's H heads over all S tokens (q, k, v as for h3s_attention) with the inverse exchange in
 * its epilogue: the output row of token t is stored straight into rank t / (S/P)'s token shard out_shards[t / (S/P)]
 * [S/P, P*H*D] (out_dt; this rank's own buffer or one opened with h3s_ipc_open) at row t % (S/P), columns
 * rank*H*D .. rank*H*D + H*D - 1. No separate output pass; the ranks must meet before another rank reads its shard. */
int h3s_attention_ulysses(void* ctx, const void* q, const void* k, const void* v, int dt, int64_t S, int64_t H,
                          int64_t D, int64_t stride, void* const* out_shards, int P, int rank, int out_dt);

/* The Sage pre-pass alone (kernels/h3sycl.cpp:1733-1761 as a callable step, for parity checks and for callers that
 * keep int8 q/k): iq, ik int8 [H, S, D]; sc float [2*H*nb + H*D] = q scales [H, nb], k scales [H, nb], k's channel
 * mean [H*D], nb = ceil(S / 64). D = 64 or 128. Queued on the context's stream. */
int h3s_sage_prepass(void* ctx, const void* q, const void* k, int dt, int64_t S, int64_t H, int64_t D, int64_t stride,
                     int8_t* iq, int8_t* ik, float* sc);
/* h3s_rms_rope(q, wq), h3s_rms_rope(k, wk), then h3s_sage_prepass, in one call with the same results bit for bit (q
 * and k are left normalised and rotated in place, as the two calls leave them). eps, cs and rot_dim as h3s_rms_rope,
 * with its refusals; D = 64 or 128, as h3s_sage_prepass. */
int h3s_sage_prepass_rope(void* ctx, void* q, void* k, int dt, int64_t S, int64_t H, int64_t D, int64_t stride,
                          const float* wq, const float* wk, float eps, const float* cs, int rot_dim, int8_t* iq,
                          int8_t* ik, float* sc);
/* A denoiser block's three calls before its output projection (engine/h3-core/src/dit.rs:347-350), in one:
 * h3s_rms_rope(q, wq), h3s_rms_rope(k, wk), h3s_attention(q, k, v, ..., out). The Sage path runs the fused pre-pass
 * above; the fp16 SDPA path normalises q and k first. q and k are left normalised and rotated in place either way;
 * the output is h3s_attention's on those rows. The refusals of both calls. */
int h3s_attention_rms_rope(void* ctx, void* q, void* k, const void* v, int dt, int64_t S, int64_t H, int64_t D,
                           int64_t stride, void* out, int out_dt, const float* wq, const float* wk, float eps,
                           const float* cs, int rot_dim);
/* The CUDA stream a context queues on (a cudaStream_t), for callers that order their own work with it. */
void* h3s_stream(void* ctx);
/* Self-test of the kernels' bounded waits: queues a kernel that waits `wait_ns` nanoseconds for an mbarrier nothing
 * arrives at, gives up, and records the failure like any kernel of this library; the following h3s_wait returns -1.
 * It faults nothing and leaves the context usable. */
int h3s_selftest_wait_timeout(void* ctx, uint64_t wait_ns);

/* The int8 Sage attention with no device allocation at all. No counterpart in the reference. For callers that cannot
 * allocate device memory when they call: code on a path that must not synchronise the device (cudaMalloc and cudaFree
 * may), and hosts whose device memory is wholly owned and budgeted by another allocator (a fixed cap, a caching
 * allocator), where a library allocating behind their back breaks the budget.
 * It computes what h3s_attention computes on its Sage path (K channel mean, int8 q/k per 64-row block, the tcgen05
 * kernel) for fp16 q, k, v rows at `stride` (16-byte aligned starts, stride a multiple of 8), D = 128, into out
 * [S, H*D] in out_dt, queued on *stream (stream points to a cudaStream_t; NULL: the legacy default stream). Its scratch
 * is a fixed array of 8 MiB + 128 KiB inside this library, which every GPU that loads the library holds until the
 * process exits: S*H*D <= 4,194,304 and H*D <= 16,384, else -1 with the limit in h3s_last_error(). The first call on
 * a device looks the array's address up (cudaGetSymbolAddress); make that first call before any stream capture.
 * err: a device int of the caller; each call first sets it to 0 on the stream, and a kernel whose wait gives up ORs a
 * nonzero code into it. Each GPU has its own copy of the array, shared by every call on that GPU: two calls on one GPU
 * whose work overlaps (different streams, not ordered by events) race on it, so order them. */
int h3s_attention_sage_static(void* stream, const void* q, const void* k, const void* v, int64_t S, int64_t H, int64_t D,
                              int64_t stride, void* out, int out_dt, int* err);

/* ---- the text model token by token: an 8-bit key/value cache and 4-bit linear layers ------------------------------ */

/* No counterpart in the reference, whose text encoder reads a whole prompt at once (h3s_attention_causal). These serve
 * a text model with grouped heads over sequences that grow. None of them allocates or waits for anything, so a CUDA
 * graph can hold them; the lengths, tables and counts that they go by live on the device and may change between
 * replays. Scratch is the caller's (work).
 *
 * The cache of `seqs` sequences: pages of 64 tokens with one float scale per page and head, in a pool that the sequences
 * share through `table`; the tokens of a sequence that do not fill a page yet are in its tail, in the rows' own type dt.
 * Token (slot) s of sequence b, head h: s < 64 * (lens[b] / 64): page table[b, s / 64], value code * scale, in float;
 * else tail row s % 64. Which pages are free is the caller's to keep. A page id outside the pool, or lens / starts out
 * of range, is found by the kernels: that page counts as unseen (attention) or is not written (append), that sequence is
 * left alone (eviction; lens and starts in all of them), and the next h3s_wait returns -1. Starts that run backwards may
 * leave any row of out as it was. All arrays are contiguous; k, v, tail_k and tail_v start on 16 bytes. */
typedef struct h3s_kv_cache {
    int8_t *k, *v;             /* [pages, heads, 64, dim] codes */
    float *k_scale, *v_scale;  /* [pages, heads] */
    void *tail_k, *tail_v;     /* [seqs, heads, 64, dim] in dt */
    float* weight;             /* [pages, heads, 64] the attention weight each token has received, or NULL */
    float* tail_weight;        /* [seqs, heads, 64]; NULL with weight */
    int32_t* table;            /* [seqs, width] page ids, of which a sequence uses the first lens / 64 */
    int32_t* lens;             /* [seqs] tokens, those of the current call included */
    int64_t pages, seqs, width, heads, dim;   /* dim 64 or 128; width < 2^25 */
    int32_t dt;
} h3s_kv_cache;

/* Writes the last n = starts[b+1] - starts[b] of sequence b's lens[b] tokens, for every b: rows starts[b] ... of k and v
 * (T rows of heads x dim, row r at element r * stride, type dt; starts int32 [seqs + 1], rows behind starts[seqs] are not
 * read). A block of 64 slots that is full now goes to page table[b, slot / 64]: scale = a / 127 with a the largest finite
 * magnitude of its 64 x dim values of a head, code = 127 x / a rounded to the nearest, half way to even (the exact ratio;
 * an infinity takes +-127, a NaN 0). The rest goes to the tail, so that the result does not depend on how the tokens
 * were spread over calls. A page that is written takes over its tokens' weights; a new token's is 0. max_new: what the
 * largest n is about (0: T), for the division of the work; no n is wrong. */
int h3s_kv_append(void* ctx, const h3s_kv_cache* kv, const void* k, const void* v, int64_t T, int64_t stride,
                  const int32_t* starts, int64_t max_new);

/* Causal attention with grouped heads over the cache: query row starts[b] + i (i < n; T rows of Hq x dim at stride qs,
 * type dt) is token lens[b] - n + i of sequence b and sees the slots up to its own; query head h reads key/value head
 * h / (Hq / heads), scores q.k / sqrt(dim). out [T, Hq * dim] in dt; a row that sees nothing (lens[b] < n) is 0, rows
 * behind starts[seqs] are left as they were. An infinite or NaN value in the tail (a page's codes have none) makes its
 * feature infinite or NaN in every row that sees it, however small its weight. Scores, the softmax's maximum and sums and the
 * sums of weighted values are held in float (these without the division: a value's size times a sequence's tokens stays
 * below 2^113). What enters the products in fewer bits are the softmax's weights, as fp16 with a power of two per row for a
 * 16-bit dt (off by up to 2^-11 of each) and as two fp16 terms for float32, and float32 queries, as two fp16 terms (2^-22).
 * out is rounded once to dt. accumulate: weight[slot] += the sum of the slot's softmax weights over the rows and heads that
 * read it (kv->weight needed; in any order for a page that sequences share). It scores the keys a second time, in a form
 * made for single tokens: a long prompt takes several times as long with it. max_new, max_len: what the largest n and length
 * are about (0: T, 64 * width), for the division of the work; none is wrong. work: work_bytes of device memory, at least
 * h3s_attention_cached_work(...) of the same arguments, on 16 bytes, this call's own until it has run. */
int h3s_attention_cached(void* ctx, const h3s_kv_cache* kv, const void* q, int64_t T, int64_t Hq, int64_t qs,
                         const int32_t* starts, int64_t max_new, int64_t max_len, void* out, int accumulate, void* work,
                         uint64_t work_bytes);
uint64_t h3s_attention_cached_work(void* ctx, const h3s_kv_cache* kv, int64_t T, int64_t Hq, int64_t max_new,
                                   int64_t max_len, int accumulate);

/* Cuts every sequence longer than `budget` (a multiple of 64) to it. Each head keeps its own tokens: the first `sinks`,
 * the last `recent`, and of the others those with the largest weight (of equal ones the earlier; a NaN counts least), in
 * their order. They are quantised again, as h3s_kv_append does, into the pages spare [seqs, budget / 64], weights with
 * them; then the first budget / 64 entries of the sequence's table and of its row of spare change places, and lens[b] =
 * budget: the old pages are the next eviction's spare ones. Sequences up to the budget keep everything, spare included.
 * A spare page belongs to no sequence and is named once, and so must an evicted sequence's old pages be: one that another
 * table names too (a common prefix) would be written over by the next eviction. work: 4 * seqs * heads * budget bytes. */
int h3s_kv_evict(void* ctx, const h3s_kv_cache* kv, int32_t* spare, int64_t budget, int64_t sinks, int64_t recent,
                 void* work, uint64_t work_bytes);

/* A linear layer with 4-bit weights for a few rows of x, out = x . W^T + bias:
 *   W[n, k] = scale[k / group, n] * (code[n, k] - zero[k / group, n])      code 0..15, zero NULL: 8
 * x [M, K] in x_dt; scale and zero [ceil(K / group), N] in s_dt; bias float [N] or NULL; out [M, N] in out_dt, rounded
 * once from float. Sums are taken in float, as sum x (code - 8) + (8 - zero) sum x, and scaled per group; one that is not
 * finite is taken again, term by term in 64 bits, so that infinities and NaN come out as the definition has them, and what
 * passes float's largest only on its way as it is (an output of this kind costs a pass of one thread over its K terms).
 * group 32, 64, 128 or 0 (one scale per output). tiles: the codes as h3s_int4_pack lays them out, 16 * ceil(N / 16) * 64 *
 * ceil(K / 64) / 2 bytes on 16 bytes. Any M up to 2,097,120 is right (from some hundred rows on a matrix product on unpacked
 * weights is faster); N up to 2^29 - 128, K up to 2^30; more is refused. M, K or N <= 0: nothing to do, returns 0. */
int h3s_int4_linear(void* ctx, const void* x, int x_dt, int64_t M, int64_t K, const void* tiles, int64_t N,
                    const void* scale, const void* zero, int s_dt, int group, const float* bias, void* out, int out_dt);
/* codes uint8 [N, K / 2] (K even), input 2 i in the low four bits of byte i -> tiles, once per layer. */
int h3s_int4_pack(void* ctx, const uint8_t* codes, int64_t N, int64_t K, void* tiles);

#ifdef __cplusplus
}
#endif
#endif
