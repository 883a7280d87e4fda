#pragma once
// hipgpt_attn.h -- C ABI of the MI355X attention forward library
// (libhipgpt_attn.so).  Plain pointers and sizes; no C++ or torch types.
//
// Every entry point is asynchronous on the given stream (0 = null stream),
// allocates nothing unless stated, and returns HIPGPT_OK or a negative
// status (see hipgpt_attn_strerror).  Pointers are device pointers.

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    HIPGPT_OK = 0,
    HIPGPT_ERR_INVALID = -1,      /* bad size, stride, pointer or flag        */
    HIPGPT_ERR_UNSUPPORTED = -2,  /* valid problem this build has no kernel for */
    HIPGPT_ERR_LAUNCH = -3,       /* the HIP launch itself failed             */
    HIPGPT_ERR_WORKSPACE = -4,    /* workspace missing or too small           */
    HIPGPT_ERR_SCRATCH = -5       /* beyond the no-allocation entry's scratch */
};

enum { HIPGPT_F32 = 0, HIPGPT_BF16 = 1 };

/* Output layouts of hipgpt_qkv_projection. */
enum { HIPGPT_QKV_ROWS = 0, HIPGPT_QKV_PLANAR = 1 };

/* Text for a status code. */
const char* hipgpt_attn_strerror(int status);

/* C-linkage twin of launch_multihead_attention (include/hip_kernels.h), for
 * FFI callers that cannot bind a C++ symbol.  Same contract, including the
 * abort on H <= 0 or E % H != 0.  Replaces src/hip_kernels.cpp:404-451. */
void hipgpt_launch_multihead_attention(const float* d_qkv, float* d_output,
                                       float* d_attn_probs, int B, int S,
                                       int E, int H);

/* C-linkage twins of HipGPT's unfused helpers (include/hip_kernels.h:44-46),
 * same contract as the C++ symbols declared in include/hip_kernels.h. */
void hipgpt_launch_scaled_dot_product(const float* Q, const float* K,
                                      float* scores, int B, int S, int D);
void hipgpt_launch_softmax(const float* scores, float* softmax_out, int B,
                           int S);
void hipgpt_launch_attention_weighted_sum(const float* softmax, const float* V,
                                          float* output, int B, int S, int D);

/* C-linkage twin of launch_multihead_attention_backward
 * (include/hip_kernels.h; replaces src/hip_kernels.cpp:1159-1272). */
void hipgpt_launch_multihead_attention_backward(const float* d_grad_attn_output,
                                                const float* d_qkv,
                                                const float* d_softmax,
                                                float* d_grad_qkv, int B, int S,
                                                int E, int H);

/* Backward with a caller-owned workspace (hipgpt_attn_bwd_workspace_bytes:
 * B*H*S floats), a stream, and a causal flag that skips tiles of the probs
 * wholly above the diagonal (a causal forward wrote zeros there).  Same
 * buffers as the drop-in; returns a status. */
size_t hipgpt_attn_bwd_workspace_bytes(int B, int S, int H);
int hipgpt_attn_bwd_qkv_planar(const float* grad_out, const float* qkv,
                               const float* probs, float* grad_qkv, int B,
                               int S, int E, int H, int causal,
                               void* workspace, size_t workspace_bytes,
                               hipStream_t stream);

/* No counterpart in HipGPT.  hipgpt_attn_bwd_qkv_planar without a workspace
 * argument, for callers that cannot allocate: code under HIP graph capture,
 * tight serving/training loops, harnesses that forbid hipMalloc.  It calls no
 * allocator; its B*H*S row-dot workspace is a fixed 4 MiB array per GPU
 * inside the library, so B*H*S must be at most 1048576 (else
 * HIPGPT_ERR_SCRATCH, nothing launched).  Calls that overlap on one GPU (two
 * streams, or host threads) share that array and race; serialise them.
 * Results are identical to hipgpt_attn_bwd_qkv_planar's. */
int hipgpt_attn_bwd_qkv_planar_noalloc(const float* grad_out, const float* qkv,
                                       const float* probs, float* grad_qkv,
                                       int B, int S, int E, int H, int causal,
                                       hipStream_t stream);

/* Training pair without the [B][H][S][S] probs buffer (FlashAttention-2's
 * forward/backward split).  No counterpart in HipGPT, whose backward reads the
 * stored probs (src/hip_kernels.cpp:1159-1272); this pair computes the same
 * gradients from O and a per-row log-sum-exp instead.
 *   forward:  planar buffers as hipgpt_attn_qkv_planar, plus
 *             lse [B][H][S] = ln sum_j exp(q_i . k_j / sqrt(D)) over the keys
 *             query i sees (all, or j <= i when causal).
 *   backward: grad_out, qkv, the forward's out and lse -> every element of
 *             the planar grad_qkv [dQ|dK|dV]; P is recomputed per tile.
 *             At D = 32 and 64 workspace / workspace_bytes are ignored (may
 *             be NULL / 0); other head dims need the B*H*S floats of
 *             hipgpt_attn_bwd_workspace_bytes (else HIPGPT_ERR_WORKSPACE).
 * fp32, D = E/H a multiple of 4 up to 256, 16-byte aligned buffers; other
 * shapes return HIPGPT_ERR_UNSUPPORTED. */
int hipgpt_attn_fwd_lse_qkv_planar(const float* d_qkv, float* d_output,
                                   float* lse, int B, int S, int E, int H,
                                   int causal, hipStream_t stream);
int hipgpt_attn_bwd_lse_qkv_planar(const float* grad_out, const float* qkv,
                                   const float* out, const float* lse,
                                   float* grad_qkv, int B, int S, int E, int H,
                                   int causal, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream);

/* HipGPT's planar [3][B*S][E] layout with the options the legacy symbol
 * lacks: causal masking (keys j <= i; probs written 0 above the diagonal so
 * HipGPT's backward, src/hip_kernels.cpp:1162-1243, stays exact) and a
 * stream.  Returns a status instead of aborting. */
int hipgpt_attn_qkv_planar(const float* d_qkv, float* d_output,
                           float* d_attn_probs, int B, int S, int E, int H,
                           int causal, hipStream_t stream);

/* General strided attention forward.
 *   q, k, v: element (b, s, h, d) at X[b*x_bs + s*x_ts + h*x_hs + d], in
 *            `dtype` (HIPGPT_F32 or HIPGPT_BF16); d is contiguous.
 *   o:       fp32, same indexing with o_* strides.
 *   probs:   optional dense fp32 [B][H][Sq][Sk] normalised probabilities.
 *   scale:   softmax scale; <= 0 selects 1/sqrt(D).
 *   causal:  query i sees keys j <= i + (Sk - Sq); requires Sk >= Sq.
 * fp32 inputs keep every bit: up to D = 128 each operand is split exactly into
 * three bf16 terms, six bf16 MFMAs make a product (off by at most 2^-24 of
 * itself) and sums are fp32; results that are not finite that way (infinities,
 * NaN, operands of 2^103, sums of 2^80 and more) are formed again on fp32 MFMA.
 * The backward (D <= 128) and the projections do the same.  At D <= 128 o may be q.
 * bf16 inputs are computed with bf16 MFMA and fp32 accumulation, D in
 * {32, 64, 128}, 16-byte aligned rows (strides multiple of 8). */
int hipgpt_attn_fwd(const void* q, const void* k, const void* v, float* o,
                    float* probs, int B, int H, int Sq, int Sk, int D,
                    int64_t q_bs, int64_t q_ts, int64_t q_hs,
                    int64_t k_bs, int64_t k_ts, int64_t k_hs,
                    int64_t v_bs, int64_t v_ts, int64_t v_hs,
                    int64_t o_bs, int64_t o_ts, int64_t o_hs,
                    float scale, int causal, int dtype, hipStream_t stream);

/* Single-query decode step: q [B][1][..] attends to kv_len keys (all
 * visible).  Split-KV: num_splits partial workgroups per (b, h) write
 * (max, sum, O) to `workspace`, a reduce kernel merges them.
 * num_splits <= 0 picks hipgpt_attn_decode_default_splits().  fp32, D in
 * {32, 64, 128, 256}, 16-byte aligned rows.  The workspace is caller-owned
 * device memory of hipgpt_attn_decode_workspace_bytes() bytes (may be NULL
 * when the split count is 1). */
int hipgpt_attn_decode_default_splits(int B, int H, int kv_len);
size_t hipgpt_attn_decode_workspace_bytes(int B, int H, int D, int num_splits);
int hipgpt_attn_decode(const float* q, const float* k, const float* v,
                       float* o, int B, int H, int kv_len, int D,
                       int64_t q_bs, int64_t q_hs,
                       int64_t k_bs, int64_t k_ts, int64_t k_hs,
                       int64_t v_bs, int64_t v_ts, int64_t v_hs,
                       int64_t o_bs, int64_t o_hs,
                       float scale, int num_splits, void* workspace,
                       size_t workspace_bytes, hipStream_t stream);

/* One KV-cached decode step for a batch of sequences of different lengths
 * (the step HipGPT's generation loop, src/gpt_model.cpp:261-273, would take
 * instead of recomputing the whole window per token).
 *   k_cache, v_cache: [B][max_len][H][D] fp32, element (b, t, h, d) at
 *     X[b*c_bs + t*c_ts + h*c_hs + d]; rows [0, lens[b]) hold the cached
 *     keys / values of sequence b.
 *   lens: device int32 [B], read on the device (no host synchronisation).
 *   q, k_new, v_new, o: the step's rows [B][H][D] with (bs, hs) strides.
 * The step writes k_new / v_new into row lens[b] of the caches, computes
 * o = softmax(q K^T * scale) V over the lens[b] + 1 rows, and, when advance
 * is non-zero, increments lens[b].  A sequence with lens[b] < 0 or
 * lens[b] >= max_len is left unchanged and gets a NaN output.  Split-KV as
 * hipgpt_attn_decode (num_splits <= 0 picks the default for max_len; the
 * workspace is hipgpt_attn_decode_workspace_bytes(B, H, D, splits)).  fp32,
 * D in {32, 64, 128, 256}, 16-byte aligned rows.  Rows past lens[b] + 1 are
 * never read. */
int hipgpt_attn_decode_kvcache(const float* q, const float* k_new,
                               const float* v_new, float* k_cache,
                               float* v_cache, int* lens, float* o, int B,
                               int H, int D, int max_len,
                               int64_t q_bs, int64_t q_hs,
                               int64_t kn_bs, int64_t kn_hs,
                               int64_t vn_bs, int64_t vn_hs,
                               int64_t c_bs, int64_t c_ts, int64_t c_hs,
                               int64_t o_bs, int64_t o_hs, float scale,
                               int num_splits, int advance, void* workspace,
                               size_t workspace_bytes, hipStream_t stream);

/* ---- paged key/value cache in 8 bits ----
 * No counterpart in HipGPT.  Keys and values live in pages of `page_size`
 * tokens (32, 64 or 128) of one sequence, as codes u = c + 128 (c a whole
 * number in [-127, 127]) with one fp32 scale per (page, head) for K and one
 * for V; a value is c * scale.  heads: the cached heads; query heads are a
 * multiple of them, query head x reads cached head x / (Hq / heads).
 * head_dim D in {32, 64, 128, 256}.
 *   k, v:    element (page, head) at X + page * page_stride + head *
 *            head_stride, page_size * D bytes each; 16-byte aligned, strides
 *            multiples of 16.  All heads of a page lie within a page_stride,
 *            or all pages of a head within a head_stride.
 *            K is [token][D]; V is [token / 32][D / 32][4]
 *            [16][2][2][4], where token % 32 = 16 i3 + 4 i0 + i4 and d % 32 =
 *            16 i2 + i1 of the last five indexes i0 .. i4.
 *   scales:  (page, head) at S[page * scale_page_stride + head *
 *            scale_head_stride]; 2^-126 or more, or NaN for a page that was
 *            given a value that is not finite.
 * Memory of pages that no sequence holds is never read or written. */
typedef struct hipgpt_kvq8_cache {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t page_stride, head_stride;
    int64_t scale_page_stride, scale_head_stride;
    int num_pages, page_size, heads, head_dim;
} hipgpt_kvq8_cache;

/* One step of a batch of sequences, shared by all layers.  All arrays are on
 * the device and read there (no host synchronisation).
 *   block_table: int [batch][max_pages] (row stride table_stride): the page
 *                of tokens j * page_size .. of each sequence.
 *   lens:        int [batch], tokens of each sequence, the step's new ones
 *                included.
 *   cu_new:      int [batch + 1]: sequence b's new tokens are rows cu_new[b]
 *                .. cu_new[b + 1] - 1 of the packed buffers and positions
 *                lens[b] - n .. lens[b] - 1.  NULL: one token each, row b
 *                (then T = batch and max_new = 1).  lens[b] = 0 is then an
 *                empty slot: appends and reads skip it, attention gives zeros.
 *   max_new:     the most new tokens of any sequence.
 * A sequence with lens[b] < n (any negative length: a slot without a
 * sequence), more tokens than its table holds, or n > max_new is left as it is
 * and gets NaN rows (the first max_new); so does what reads a page index
 * outside [0, num_pages), which appends skip.  Rows that no sequence names
 * (a cu_new that is not increasing or passes T) are left as they were.  Pages
 * that several sequences hold may be read by all, and appended to by none.
 * table_stride >= max_pages. */
typedef struct hipgpt_kvq8_batch {
    const int* block_table;
    int64_t table_stride;
    int* lens;
    const int* cu_new;
    int batch, max_pages, max_new;
} hipgpt_kvq8_batch;

/* Host: turns per position of the rot_dim / 2 rotated pairs, base^(-2i /
 * rot_dim) / 2 pi, as 0.64 fixed point.  base >= 1. */
int hipgpt_rope_freqs(uint64_t* freqs, int rot_dim, double base);

/* Appends the new tokens' keys and values, rotated by position on the way.
 *   q, k, v: [T] rows of Hq / heads / heads head rows in `dtype`, element
 *            (t, h, d) at X[t * x_ts + h * x_hs + d]; 16-byte aligned rows.
 *   q_out:   receives the rotated q (q itself, or memory apart from q, k and
 *            v); q and q_out NULL: none.
 *   freqs:   device [rot_dim / 2] as hipgpt_rope_freqs gives them: pair i of
 *            position p turns by p * freqs[i] (exact at any position).  The
 *            pairs are (i, i + rot_dim / 2), or (2i, 2i + 1) where
 *            interleaved; head dims from rot_dim on stay.  NULL: no rotation.
 *   advance: non-zero first raises lens[b] by the sequence's new tokens (the
 *            first layer's append of a step), negative ones apart; 0: lens
 *            includes them already.
 * Per (page, head) the new scale is max|x| / 127 over the page's new rows, at
 * least 2^-126 and, where the page holds earlier tokens, at least their scale;
 * where that grows, their codes are rounded again to the new one.  Codes are
 * rounded to nearest even. */
int hipgpt_kvq8_append(const hipgpt_kvq8_cache* cache,
                       const hipgpt_kvq8_batch* batch, int T, const void* q,
                       void* q_out, const void* k, const void* v, int Hq,
                       int64_t q_ts, int64_t q_hs, int64_t qo_ts,
                       int64_t qo_hs, int64_t k_ts, int64_t k_hs, int64_t v_ts,
                       int64_t v_hs, const uint64_t* freqs, int rot_dim,
                       int interleaved, int dtype, int advance,
                       hipStream_t stream);

/* The values that the last cu_new[b + 1] - cu_new[b] tokens of each sequence
 * stand for, packed as the append takes them, in `dtype`. */
int hipgpt_kvq8_read(const hipgpt_kvq8_cache* cache,
                     const hipgpt_kvq8_batch* batch, int T, void* k, void* v,
                     int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs,
                     int dtype, hipStream_t stream);

/* Attention over the cache.
 *   decode:  one query row per sequence (cu_new NULL), over its lens[b]
 *            tokens.  An empty slot gives zeros.
 *   prefill: the new tokens of each sequence (T rows, packed as cu_new says);
 *            the cache holds them already, token i of n sees keys
 *            j <= lens[b] - n + i.
 *   q: in `dtype`, rotated already; o: in out_dtype; element (row, h, d) at
 *   X[row * x_ts + h * x_hs + d], 16-byte aligned rows.  An fp32 q takes an
 *   fp32 o.  scale <= 0 selects 1/sqrt(D).
 * num_splits > 1 divides the work and joins the parts by a second kernel
 * through a caller-owned, 16-byte aligned workspace of
 * hipgpt_attn_kvq8_workspace_bytes: with few query rows per cached head and
 * sequence, each row's keys num_splits ways; with more, the keys of all blocks
 * of 128 rows in num_splits equal shares.  At most 1024; <= 0:
 * hipgpt_attn_kvq8_default_splits for max_len = max_pages * page_size (in
 * decode T = B and max_new = 1).  1 needs no workspace.  Calls that may run at
 * the same time, replayed graphs among them, need workspaces of their own.
 * Sums and softmax statistics are fp32.  With an fp32 result the products are
 * off by 2^-22 of themselves at most; with a bf16 result the softmax weights
 * are rounded to fp16 first.  V scales are applied to those weights relative
 * to the largest scale that the row's block of rows met, so what pages with
 * scales under 2^-24 of it contribute is lost in part (fp16's range). */
int hipgpt_attn_kvq8_default_splits(int B, int T, int max_new, int Hq,
                                    int heads, int D, int out_dtype,
                                    int max_len);
size_t hipgpt_attn_kvq8_workspace_bytes(int B, int T, int max_new, int Hq,
                                        int heads, int D, int out_dtype,
                                        int num_splits);
int hipgpt_attn_decode_kvq8(const hipgpt_kvq8_cache* cache,
                            const hipgpt_kvq8_batch* batch, const void* q,
                            void* o, int Hq, int64_t q_ts, int64_t q_hs,
                            int64_t o_ts, int64_t o_hs, float scale, int dtype,
                            int out_dtype, int num_splits, void* workspace,
                            size_t workspace_bytes, hipStream_t stream);
int hipgpt_attn_prefill_kvq8(const hipgpt_kvq8_cache* cache,
                             const hipgpt_kvq8_batch* batch, int T,
                             const void* q, void* o, int Hq, int64_t q_ts,
                             int64_t q_hs, int64_t o_ts, int64_t o_hs,
                             float scale, int dtype, int out_dtype,
                             int num_splits, void* workspace,
                             size_t workspace_bytes, hipStream_t stream);

/* Diagnostics, no counterpart in HipGPT.  One kernel synchronises its waves
 * through LDS flags instead of barriers (the one-workgroup-per-(b, h) backward
 * from lse at D = 32, S <= 256).
 * Its waits are bounded so a fault in the schedule cannot hang the GPU; a
 * wait that runs out is counted on the device.  *count receives the number
 * of expired waits on the current device since the last clear (zero in a
 * correct run; non-zero means some outputs may be wrong).  clear != 0 resets
 * the count in the same device-side atomic that reads it.  Blocking: a
 * one-thread kernel and a copy on the null stream.  The count is exact only
 * when no library kernel is in flight on another stream (the null stream does
 * not wait for non-blocking streams): synchronise the device first. */
int hipgpt_attn_wait_expired(unsigned int* count, int clear);

/* ---- projections either side of the attention ---- */

/* C-linkage twins of launch_matmul / launch_matmul_add_bias
 * (include/hip_kernels.h; replace src/hip_kernels.cpp:70-154). */
void hipgpt_launch_matmul(const float* A, const float* B, float* C, int M,
                          int N, int K);
void hipgpt_launch_matmul_add_bias(const float* A, const float* B,
                                   const float* bias, float* C, int M, int N,
                                   int K);

/* General GEMM + bias: C[m][n] = sum_k A[m][k] W[k][n] (+ bias[n]).
 *   A [M][K] row stride lda; W [K][N] row stride ldw; bias [N] or NULL.
 *   Output column n is stored at C + (n / seg_w) * seg_stride + m * ldc
 *   + n % seg_w (elements of out_dtype): seg_w = N gives a row-major [M][N]
 *   buffer; seg_w = N/3, seg_stride = M*N/3 splits a QKV projection into
 *   planar [3][M][N/3].  out_dtype HIPGPT_F32 or HIPGPT_BF16 (RNE).
 *   Requires M, N >= 1, K >= 0, lda >= K, ldw >= N, 1 <= seg_w <= N,
 *   ldc >= seg_w, seg_stride >= 0. */
int hipgpt_gemm_bias(const float* A, const float* W, const float* bias,
                     void* C, int M, int N, int K, int64_t lda, int64_t ldw,
                     int64_t ldc, int seg_w, int64_t seg_stride,
                     int out_dtype, hipStream_t stream);

/* HipGPT's QKV projection (src/transformer_layer.cpp:217): x [T][E] times
 * w_qkv [E][3E] plus b_qkv [3E].  layout HIPGPT_QKV_ROWS writes the
 * reference's [T][3E] buffer; HIPGPT_QKV_PLANAR writes [3][T][E], so that
 * plane p row t is projection p of token t in the layout the attention
 * launchers read.  out_dtype HIPGPT_F32 or HIPGPT_BF16. */
int hipgpt_qkv_projection(const float* x, const float* w_qkv,
                          const float* b_qkv, void* out, int T, int E,
                          int layout, int out_dtype, hipStream_t stream);

#ifdef __cplusplus
}
#endif
