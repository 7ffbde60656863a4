/*
 * glaucis_b200 — C ABI of the B200 (sm_100a) kernels behind the two scored
 * kernel templates of the Glaucis kernel evaluator:
 *
 *   gmm_fp8_blockwise  grouped (ragged, MoE-style) matmul with block-wise FP8
 *                      quantisation: activations 1x128 fp32 scales, weights
 *                      128x128 fp32 scales, fp32 accumulation.
 *   chunk_gla          chunked Gated Linear Attention, forward.
 *
 * Conventions shared by every entry point:
 *   - All pointers are device pointers owned by the caller.  The library
 *     borrows them for the duration of the (asynchronous) call and never
 *     frees or retains them.
 *   - `stream` is a cudaStream_t passed as void*; NULL means the legacy
 *     default stream.  Every call is stream-ordered and returns before the
 *     GPU work finishes.
 *   - `err_word` is an optional device int.  Kernels write a non-zero
 *     GL_DEV_* code there when a bounded device-side wait gives up; pass NULL
 *     to use a per-device word owned by the library.  Read it back with
 *     gl_device_status().
 *   - Return value: GL_OK (0) on a successful launch, a negative GL_E* code
 *     otherwise; gl_last_error() then holds a message (per host thread).
 *
 * Each entry point names the reference interface it replaces (paths are
 * relative to the Glaucis repository, kernel-evolve = KE).
 */
#ifndef GLAUCIS_B200_H
#define GLAUCIS_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes. */
#define GL_OK 0
#define GL_EINVAL (-1)   /* bad shape, alignment or argument */
#define GL_ELAUNCH (-2)  /* CUDA launch / driver failure */
#define GL_EDEVICE (-3)  /* device error word was set */

/* Device error word codes (written by kernels). */
#define GL_DEV_OK 0
#define GL_DEV_WAIT_TIMEOUT 1   /* an mbarrier wait exceeded its poll budget */
#define GL_DEV_BAD_GROUPS 2     /* group_sizes sum exceeds M or a size < 0 */
#define GL_DEV_BAD_INDEX 3      /* a row index is past the rows (the row is skipped) */

/* Output dtypes of the grouped matmul. */
#define GL_OUT_BF16 0
#define GL_OUT_F32 1

/*
 * Block-wise activation quantiser, 1x128 tiles along K.
 *   x  bf16 [M, K] row-major, K % 128 == 0
 *   q  e4m3fn [M, K] row-major (one byte per element)
 *   s  fp32 [M, K/128] row-major, s = absmax(block)/448 (1.0 for an all-zero
 *      block), q = round-to-nearest-even(x / s) saturated to +-448.
 * Replaces: qwix.pallas.quantize(lhs, float8_e4m3fn, channelwise_axes=[0],
 *   tiled_axes={1: 128}, calibration_method="absmax", scale_dtype=f32)
 *   called at KE/examples/kernels/gmm_fp8_blockwise.py:84-91.
 */
int gl_quant_act_1x128(const void* x, int64_t M, int64_t K, void* q, float* s,
                       int* err_word, void* stream);

/*
 * Block-wise weight quantiser, 128x128 tiles over (K, N) per group.
 *   w  bf16 [G, K, N] row-major, K % 128 == 0, N % 128 == 0
 *   q  e4m3fn [G, K, N] row-major
 *   s  fp32 [G, K/128, N/128]
 * Replaces: qwix.pallas.quantize(rhs, float8_e4m3fn, channelwise_axes=[0],
 *   tiled_axes={1: 128, 2: 128}, ...) at
 *   KE/examples/kernels/gmm_fp8_blockwise.py:100-107.
 */
int gl_quant_w_128x128(const void* w, int64_t G, int64_t K, int64_t N, void* q,
                       float* s, int* err_word, void* stream);

/*
 * Grouped matmul forward on pre-quantised operands:
 *   out[m, n] = sum_kb a_s[m, kb] * b_s[g, kb, n/128]
 *                      * sum_{k in block kb} a_q[m, k] * b_q[g, k, n]
 * where rows [off_g, off_g + group_sizes[g]) belong to group g and off_g is
 * the exclusive prefix sum of group_sizes.  Rows at or beyond
 * sum(group_sizes) are not written.
 *   a_q e4m3fn [M, K], a_s fp32 [M, K/128]      (layout of gl_quant_act_1x128)
 *   b_q e4m3fn [G, K, N], b_s fp32 [G, K/128, N/128] (gl_quant_w_128x128)
 *   group_sizes int32 [G] (device), out [M, N] bf16 or fp32 (out_dtype).
 *   K % 128 == 0, N % 128 == 0, 1 <= G <= 1024.
 * Replaces: tokamax pallas_mosaic_tpu_kernel.gmm(lhs=QArray, rhs=QArray,
 *   group_sizes, out_dtype=f32, transpose_rhs=False) at
 *   KE/examples/kernels/gmm_fp8_blockwise.py:109-119 (reference oracle:
 *   KE/examples/kernels/gmm_fp8_blockwise_ref.py:67-77).
 */
int gl_gmm_fp8_fwd(const void* a_q, const float* a_s, const void* b_q,
                   const float* b_s, const int32_t* group_sizes, int64_t G,
                   int64_t M, int64_t K, int64_t N, void* out, int out_dtype,
                   int* err_word, void* stream);

/* Largest n_outs of gl_gmm_fp8_fwd_scatter. */
#define GL_MAX_SCATTER_OUTS 8

/*
 * gl_gmm_fp8_fwd with its output rows stored into several buffers: row m of
 * this call is written as row row_offset + m of each of outs[0 .. n_outs-1]
 * (each at least row_offset + M rows of N elements of out_dtype, 16-byte
 * aligned).  The buffers may be other GPUs' memory mapped into this process
 * (CUDA IPC peer mappings over NVLink, e.g. gl_ipc_open): the kernel only
 * stores to them (bf16: TMA stores of each finished 32-row slice from shared
 * memory; fp32 and a group's last rows: direct stores), so a grouped matmul
 * sharded by expert group across ranks assembles the full output on every
 * rank inside its epilogue, overlapped with the MMAs, instead of an
 * all-gather after it.  The caller
 * orders the readers after the kernels of all ranks (a barrier).  Rows past
 * sum(group_sizes) are not written.  No counterpart in the reference (its
 * sharded output would be all-gathered by a collective).
 */
int gl_gmm_fp8_fwd_scatter(const void* a_q, const float* a_s, const void* b_q, const float* b_s,
                           const int32_t* group_sizes, int64_t G, int64_t M, int64_t K, int64_t N,
                           void* const* outs, int n_outs, int64_t row_offset, int out_dtype,
                           int* err_word, void* stream);

/*
 * Peer buffers for gl_gmm_fp8_fwd_scatter across processes (one per GPU):
 * gl_ipc_alloc allocates device memory on the current device and returns its
 * CUDA IPC handle (GL_IPC_HANDLE_BYTES bytes); another process opens it with
 * gl_ipc_open (a unicast peer mapping over NVLink; no multicast object) and
 * releases the mapping with gl_ipc_close; the owner frees with gl_ipc_free.
 */
#define GL_IPC_HANDLE_BYTES 64
int gl_ipc_alloc(size_t bytes, void** ptr, void* handle);
int gl_ipc_open(const void* handle, void** ptr);
int gl_ipc_close(void* ptr);
int gl_ipc_free(void* ptr);

/*
 * Chunked Gated Linear Attention forward (fixed-length sequences).
 *   q, k  bf16 [B, T, H, K];  v bf16 [B, T, H, V];  K == 128, V == 128
 *   g       fp32 [B, T, H, K] per-key log-gate (raw, not cumsummed) or NULL
 *   g_gamma fp32 [H] per-head constant log-gate or NULL (exactly one of
 *           g / g_gamma must be non-NULL)
 *   h0      fp32 [B, H, K, V] initial state or NULL (zeros)
 *   o       bf16 [B, T, H, V] output
 *   ht      fp32 [B, H, K, V] final state or NULL (not written)
 *   chunk_size == 64, T % 64 == 0.
 * Semantics: within each chunk G = cumsum(g) (chunk-local);
 *   o = scale*(q*e^G) h_n + tril(scale*(q*e^G)(k*e^-G)^T) v
 *   h_{n+1} = e^{G_last} * h_n + (k*e^{G_last-G})^T v.
 * Replaces: chunk_gla_fwd(q, k, v, g_gamma, scale, chunk_size) at
 *   KE/examples/kernels/chunk_gla.py:258-273 (three pallas_calls
 *   chunk_fwd_h :94-138, chunk_gla_fwd_intra_gk :163-188,
 *   chunk_gla_fwd_o_gk :218-250), with the per-key gate / h0 / final-state
 *   semantics of chunk_fwd_h_ref at
 *   KE/upstream/fused_chunk_simple_gla/common_chunk_h.py:363-489.
 */
int gl_chunk_gla_fwd(const void* q, const void* k, const void* v, const float* g,
                     const float* g_gamma, const float* h0, float scale,
                     int64_t B, int64_t T, int64_t H, int64_t K, int64_t V,
                     int64_t chunk_size, void* o, float* ht, int* err_word,
                     void* stream);

/* Flags of gl_chunk_gla_fwd_ex. */
#define GL_GLA_BF16_INTRA 1  /* tril(A) v with A rounded to bf16 once (see below) */

/*
 * The chunked GLA forward with every option: gl_chunk_gla_fwd_ws (h_states
 * NULL) or gl_chunk_gla_fwd_states (h_states non-NULL) plus `flags`.
 *   flags = 0 (also every other gl_chunk_gla_fwd* entry point): the
 *     intra-chunk product tril(A) v = P_hi v + P_lo v with P_hi =
 *     bf16(tril(A)) and P_lo = bf16(tril(A) - P_hi), so A enters the product
 *     to ~2^-17 relative, as the template's output kernel multiplies fp32 A
 *     by v at Precision.HIGHEST (KE/examples/kernels/chunk_gla.py:208-212).
 *   flags = GL_GLA_BF16_INTRA: A rounded to bf16 once on the tensor core
 *     (fp32 accumulation), the operand precision of the reference's jnp
 *     oracle at default matmul precision on its TPU platform
 *     (KE/examples/kernels/chunk_gla_ref.py:96-97); about 10 % faster.
 * Replaces chunk_gla_fwd (KE/examples/kernels/chunk_gla.py:258-273) as
 * gl_chunk_gla_fwd does.
 */
int gl_chunk_gla_fwd_ex(const void* q, const void* k, const void* v, const float* g,
                        const float* g_gamma, const float* h0, float scale, int64_t B, int64_t T,
                        int64_t H, int64_t K, int64_t V, int64_t chunk_size, void* o, float* ht,
                        void* h_states, void* workspace, size_t workspace_bytes, int flags,
                        int* err_word, void* stream);

/*
 * gl_chunk_gla_fwd_ex (h_states NULL) with o stored into several buffers:
 * outs[0 .. n_outs-1], each of o's layout [B, T, H, V] bf16 and 16-byte
 * aligned, receive the same output.  The buffers may be other GPUs' memory
 * mapped into this process (CUDA IPC peer mappings over NVLink, e.g.
 * gl_ipc_open): the forward stores each chunk's O from shared memory with TMA
 * stores into every buffer, so a forward sharded by head across ranks
 * assembles its output on every rank inside the kernel instead of an
 * all-gather after it.  Needs the full-width kernel, i.e. a workspace when
 * B*H*2 <= the SM count (GL_EINVAL otherwise).  The caller orders the
 * readers after the kernels of all ranks.  No counterpart in the reference
 * (chunk_gla.py:258-273 writes one o; a head-sharded caller would all-gather).
 */
int gl_chunk_gla_fwd_scatter(const void* q, const void* k, const void* v, const float* g,
                             const float* g_gamma, const float* h0, float scale, int64_t B,
                             int64_t T, int64_t H, int64_t K, int64_t V, int64_t chunk_size,
                             void* const* outs, int n_outs, float* ht, void* workspace,
                             size_t workspace_bytes, int flags, int* err_word, void* stream);

/*
 * The intermediates of the chunked GLA forward that gl_chunk_gla_fwd keeps on
 * chip, for callers that read them:
 *   g_cumsum fp32 [B, T, H, K]  chunk-local cumsum of g (or g_gamma[h]*(1..64))
 *   A        fp32 [B, T, H, 64] A[i, j] = scale * sum_k q[i,k] e^{G[i,k]}
 *                               k[j,k] e^{-G[j,k]} per chunk, full 64x64
 *                               square (not causally masked)
 * Either output may be NULL (not written); q, k, g / g_gamma, scale and the
 * shapes as gl_chunk_gla_fwd.  fp32 arithmetic (not the tensor cores), one
 * extra pass over q, k and g.  err_word is accepted for symmetry and never
 * written (the kernel has no device-side waits).
 * Replaces the g_cumsum and A outputs of chunk_gla_fwd
 * (KE/examples/kernels/chunk_gla.py:258-273; A from chunk_gla_fwd_intra_gk
 * :146-188, g_cumsum :265-267).
 */
int gl_chunk_gla_fwd_intermediates(const void* q, const void* k, const float* g,
                                   const float* g_gamma, float scale, int64_t B, int64_t T,
                                   int64_t H, int64_t K, int64_t chunk_size, float* g_cumsum,
                                   float* A, int* err_word, void* stream);

/*
 * gl_chunk_gla_fwd with a caller-owned device workspace.  When B*H is small
 * against the SM count (few heads, long sequences) the sequence is split into
 * segments.  The first, short segment runs its full pass from h0 beside a
 * state-only pass that computes each middle segment's final state from a
 * zero state, and its total decay, into the workspace; the full pass of the
 * remaining segments then starts each of them from h0 folded with the
 * preceding segments' records, so the recurrence runs on one CTA per SM
 * instead of one per (batch, head).  The first phase forks a library-owned
 * stream from `stream` and joins it back with events.
 * gl_chunk_gla_fwd_workspace_bytes gives the size the split wants on the
 * current device (0: no split for this shape); a smaller workspace gives
 * fewer segments, NULL / 0 none.  The workspace must be 256-byte aligned and
 * not be used by another call in flight.  gl_chunk_gla_fwd is this call with
 * no workspace.  No reference counterpart: the reference scans the sequence
 * once per (batch, head) (KE/examples/kernels/chunk_gla.py:94-138).
 */
size_t gl_chunk_gla_fwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t K,
                                        int64_t V, int64_t chunk_size);
int gl_chunk_gla_fwd_ws(const void* q, const void* k, const void* v, const float* g,
                        const float* g_gamma, const float* h0, float scale,
                        int64_t B, int64_t T, int64_t H, int64_t K, int64_t V,
                        int64_t chunk_size, void* o, float* ht, void* workspace,
                        size_t workspace_bytes, int* err_word, void* stream);

/*
 * Training forward of the chunked GLA: gl_chunk_gla_fwd_ws that also writes
 * the state before every chunk, h_states bf16 [B, T/64, H, K, V]
 * (h_states[:, n] = h_n, h_0 = h0), the residual the backward reads.
 * Replaces the h output of chunk_gla_fwd (KE/examples/kernels/chunk_gla.py
 * :258-273, kept fp32 there and cast to bf16 where the backward uses it,
 * :356-359).
 */
int gl_chunk_gla_fwd_states(const void* q, const void* k, const void* v, const float* g,
                            const float* g_gamma, const float* h0, float scale,
                            int64_t B, int64_t T, int64_t H, int64_t K, int64_t V,
                            int64_t chunk_size, void* o, float* ht, void* h_states,
                            void* workspace, size_t workspace_bytes, int* err_word,
                            void* stream);

/*
 * Backward of the chunked GLA: dq, dk, dv (bf16, shaped as q, k, v) and,
 * when dh0 is non-NULL, the gradient of the initial state (fp32 [B,H,K,V]),
 * for the loss sum(o * dout) (+ sum(ht * dht) when dht is non-NULL).
 *   h_states  the forward's bf16 [B, T/64, H, K, V] (gl_chunk_gla_fwd_states)
 *   dout      bf16 [B, T, H, V];  dht fp32 [B, H, K, V] or NULL
 *   g / g_gamma, scale, shapes as the forward.  The gate is not
 *   differentiated (the reference's custom_vjp returns dq, dk, dv).
 *   workspace device memory of gl_chunk_gla_bwd_workspace_bytes(...) bytes
 *   (required, 256-byte aligned): the reverse scan's per-chunk state
 *   gradient E_n = e^{G_last(n)} dL/dh_{n+1} (bf16) and the records of its
 *   sequence split.
 * Two launches: the reverse state-gradient scan (a mode of the forward's
 * sequential kernel, with its own sequence split) and the chunk-parallel
 * dq/dk/dv kernel.  Replaces _bwd of chunk_gla (KE/examples/kernels/
 * chunk_gla.py:446-453): _chunk_bwd_dh_scan :281-305 and
 * chunk_gla_bwd_fused :313-426.
 */
size_t gl_chunk_gla_bwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t K,
                                        int64_t V, int64_t chunk_size);
int gl_chunk_gla_bwd(const void* q, const void* k, const void* v, const float* g,
                     const float* g_gamma, const void* h_states, const void* dout,
                     const float* dht, float scale, int64_t B, int64_t T, int64_t H,
                     int64_t K, int64_t V, int64_t chunk_size, void* dq, void* dk, void* dv,
                     float* dh0, void* workspace, size_t workspace_bytes, int* err_word,
                     void* stream);

/*
 * Backward of the grouped matmul (KE/examples/kernels/gmm_fp8_blockwise.py:123-169).
 *
 * gl_quant_col_128x1: 128x1 column blocks of x bf16 [M, C] (M, C multiples
 *   of 128): q e4m3 [M, C], s fp32 [M/128, C], s = absmax of 128 rows of one
 *   column / 448.  Replaces qpl.quantize(grad, channelwise_axes=[1],
 *   tiled_axes={0:128}) :135-141 and, untransposed, qpl.quantize(lhs^T,
 *   channelwise_axes=[0], tiled_axes={1:128}) :92-99 (lhs_t = (q^T, s^T)).
 * gl_gmm_fp8_dlhs: dlhs [M, K] = dout x rhs^T per group: dq / ds = dout
 *   quantised 1x128 along N (gl_quant_act_1x128 of grad [M, N]); b_q / b_s the
 *   forward's weight QArray [G, K, N] / [G, K/128, N/128].  Replaces
 *   tokamax gmm(dlhs_dout, rhs, transpose_rhs=True) :143-153.  Rows at or
 *   beyond sum(group_sizes) are not written.
 * gl_tgmm_fp8: drhs [G, K, N] = per group lhs^T x dout over the group's rows:
 *   lq / ls and dq / ds quantised by gl_quant_col_128x1 (M % 128 == 0).
 *   Empty groups get zeros.  Replaces tokamax tgmm(lhs_t, drhs_dout) :155-165.
 */
int gl_quant_col_128x1(const void* x, int64_t M, int64_t C, void* q, float* s, int* err_word,
                       void* stream);
int gl_gmm_fp8_dlhs(const void* dq, const float* ds, const void* b_q, const float* b_s,
                    const int32_t* group_sizes, int64_t G, int64_t M, int64_t K, int64_t N,
                    void* out, int out_dtype, int* err_word, void* stream);
int gl_tgmm_fp8(const void* lq, const float* ls, const void* dq, const float* ds,
                const int32_t* group_sizes, int64_t G, int64_t M, int64_t K, int64_t N,
                void* out, int out_dtype, int* err_word, void* stream);

/*
 * RMS norm with the residual's addition.  No counterpart in the reference,
 * whose templates start at the experts' products: it makes their activations.
 *   h = bf16(x + residual) (h = x when residual is NULL),
 *   r = 1 / sqrt(mean_k h^2 + eps),  y = h * r * weight
 *   x, residual  bf16 [M, K] row-major; residual may be NULL
 *   weight       [K] bf16, or fp32 with weight_f32 != 0
 *   h            bf16 [M, K], required with a residual and NULL without; may be
 *                x's or the residual's own buffer
 *   y            bf16 [M, K] or NULL
 *   q, s         e4m3fn [M, K] and fp32 [M, K/128], the layout and scales of
 *                gl_quant_act_1x128 (s = absmax(block of y)/448, 1.0 for an
 *                all-zero block), both or neither NULL, K % 128 == 0 with them;
 *                y enters them in 32 bits (not rounded to bf16 first)
 *   rstd         fp32 [M], r of every row (the backward's residual), or NULL
 * K % 8 == 0, 8 <= K <= GL_RMS_NORM_MAX_K, M <= 2^31 - 1; x, residual, weight,
 * h, y and q 16-byte aligned.  Sums are fp32.  err_word is accepted for
 * symmetry and never written (no device-side waits).
 */
#define GL_RMS_NORM_MAX_K 16384
int gl_rms_norm_fwd(const void* x, const void* residual, const void* weight, int weight_f32, float eps,
                    int64_t M, int64_t K, void* h, void* y, void* q, float* s, float* rstd,
                    int* err_word, void* stream);

/*
 * Backward of gl_rms_norm_fwd for the gradients dy of y and dh of h (dh may be
 * NULL):  u = weight * dy, xh = h * rstd,
 *   dx = rstd * (u - xh * mean_k(u * xh)) + dh   bf16 [M, K], the gradient of x
 *                                                and of the residual
 *   dweight = sum over rows of dy * xh           of weight's type, summed in
 *                                                fp32 in a fixed order
 * h, rstd as the forward wrote them (h = x without a residual).  workspace:
 * gl_rms_norm_bwd_workspace_bytes(M, K) bytes on the current device (0 for an
 * unsupported shape or M == 0), 16-byte aligned, not used by another call in
 * flight.  M == 0 gives dweight = 0.
 */
size_t gl_rms_norm_bwd_workspace_bytes(int64_t M, int64_t K);
int gl_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* weight, int weight_f32,
                    const float* rstd, int64_t M, int64_t K, void* dx, void* dweight, void* workspace,
                    size_t workspace_bytes, int* err_word, void* stream);

/* Largest topk of the router and of the exchange. */
#define GL_MOE_MAX_TOPK 32

/*
 * Router in front of the grouped matmul.  No counterpart in the reference,
 * whose templates take group_sizes as an input.
 *   logits   [T, E] fp32 (logits_f32 != 0) or bf16, 1 <= E <= 1024
 *   mask     bool [T] (one byte each, 0: the token takes no part) or NULL
 *   ids      int32 [T, topk] experts of the topk largest logits, in falling
 *            order, ties to the lowest expert; 1 <= topk <= min(E, 32)
 *   weights  fp32 [T, topk] their softmax, over its sum with renormalize != 0
 *   counts   int32 [E] choices of every expert: group_sizes of gl_gmm_fp8_fwd
 *   pos      int32 [T, topk] row of a choice when all choices are sorted by
 *            (expert, token, slot)
 *   loss     fp32 [1] balance loss E * sum_e f_e P_e, f_e = counts_e /
 *            sum(counts), P_e = the softmax's mean over the routed tokens (1
 *            when both are even; 0 without tokens)
 *   routed   fp32 [1] number of routed tokens, at least 1 (for the backward)
 * A logit of -inf takes its expert out for that token; a token that the mask
 * takes out, or whose logits are all -inf, is in no sum.  Slots without an
 * expert have ids -1, pos -1 and weight 0.  A NaN logit is never chosen, it
 * makes its token's weights and the loss NaN (so does +inf).
 * T >= 0, T * topk <= 2^31 - 1.  workspace: gl_moe_route_workspace_bytes(T, E)
 * bytes (0 when few tokens need none, or for an unsupported shape), 4-byte
 * aligned, not used by another call in flight.  err_word is accepted for symmetry and never written.
 */
size_t gl_moe_route_workspace_bytes(int64_t T, int64_t E);
int gl_moe_route_fwd(const void* logits, int logits_f32, const void* mask, int64_t T, int64_t E,
                     int64_t topk, int renormalize, int32_t* ids, float* weights, int32_t* counts,
                     int32_t* pos, float* loss, float* routed, void* workspace, size_t workspace_bytes,
                     int* err_word, void* stream);

/*
 * Backward of gl_moe_route_fwd: dlogits [T, E] (of logits' type) for the
 * gradients dweights fp32 [T, topk] and dloss fp32 [1] (device; either may be
 * NULL: zero).  logits, mask, renormalize as the forward took them, ids,
 * weights, counts and routed as it wrote them.  The choice and the counts are
 * constants.  Tokens that were not routed get zeros.
 */
int gl_moe_route_bwd(const void* logits, int logits_f32, const void* mask, const int32_t* ids,
                     const float* weights, const int32_t* counts, const float* routed,
                     const float* dweights, const float* dloss, int64_t T, int64_t E, int64_t topk,
                     int renormalize, void* dlogits, int* err_word, void* stream);

/*
 * Rows into expert order: out[pos[t, j]] = x[t] for every pos >= 0.
 *   x            [T, row_bytes] (any type; row_bytes a multiple of 16)
 *   s            fp32 [T, scales] moved alongside into out_s, or both NULL and
 *                scales 0 (with scales and T == 0, s may be NULL)
 *   pos          int32 [T, topk] as gl_moe_route_fwd writes it: the rows below
 *                sum(group_sizes), each of one choice (one that no choice names
 *                is left as it is); a negative one is skipped
 *   group_sizes  int32 [G], 1 <= G <= 1024
 *   out, out_s   [rows, ...]; rows at or past sum(group_sizes) are set to
 *                zero, their scales to 1 (the pair of a zero block)
 * A pos at or past rows is skipped and sets GL_DEV_BAD_INDEX; a negative size
 * or a sum past rows sets GL_DEV_BAD_GROUPS and leaves the tail as it is.
 * x and out 16-byte aligned; T * topk and rows <= 2^31 - 1.
 */
int gl_moe_dispatch(const void* x, int64_t row_bytes, const float* s, int64_t scales, const int32_t* pos,
                    const int32_t* group_sizes, int64_t G, int64_t T, int64_t topk, int64_t rows, void* out,
                    float* out_s, int* err_word, void* stream);

/*
 * Rows back to their tokens: out[t] = residual[t] + sum_j weights[t, j] *
 * y[pos[t, j]] over pos >= 0, summed in fp32 in slot order, rounded once.
 *   y         [rows, K] bf16, or fp32 with y_f32 != 0 (gl_gmm_fp8_fwd's out)
 *   weights   fp32 [T, topk], NULL for 1 (the backward of gl_moe_dispatch)
 *   residual  bf16 [T, K] or NULL;  out bf16 [T, K]
 * K % 8 == 0, K <= 16384; y, residual and out 16-byte aligned.  A pos past
 * rows is left out and sets GL_DEV_BAD_INDEX.
 */
int gl_moe_combine(const void* y, int y_f32, const int32_t* pos, const float* weights, const void* residual,
                   int64_t T, int64_t topk, int64_t K, int64_t rows, void* out, int* err_word, void* stream);

/*
 * Backward of gl_moe_combine for dout bf16 [T, K] (residual's gradient is dout
 * itself): dy [rows, K] of y's type, dy[pos[t, j]] = weights[t, j] * dout[t],
 * rows at or past sum(group_sizes) zero; dweights fp32 [T, topk] =
 * <dout[t], y[pos[t, j]]>, 0 where pos < 0.
 */
int gl_moe_combine_bwd(const void* dout, const void* y, int y_f32, const int32_t* pos, const float* weights,
                       const int32_t* group_sizes, int64_t G, int64_t T, int64_t topk, int64_t K,
                       int64_t rows, void* dy, float* dweights, int* err_word, void* stream);

/* Flags of gl_gmm_w4_fwd. */
#define GL_W4_ZERO_TAIL 1  /* rows at or past sum(group_sizes) are set to zero */

/*
 * Weight quantiser to 4 bits, one scale per 128 weights of a column.  No
 * counterpart in the reference.
 *   w   bf16 [G, K, N] row-major, K % 128 == 0, N % 32 == 0, G <= 1024
 *   w4  int32 [G, K/8, N]: nibble j (bits 4j..4j+3) of word [g, i, n] is
 *       q[g, 8i + j, n] + 8
 *   s   fp32 [G, K/128, N], s = absmax(128 weights)/7 (1.0 when all are zero),
 *       q = round-half-even(w / s), -7..7
 * w, w4 and s 16-byte aligned.  err_word is accepted for symmetry.
 */
int gl_quant_w4_128x1(const void* w, int64_t G, int64_t K, int64_t N, void* w4, float* s, int* err_word,
                      void* stream);

/*
 * Grouped matmul of few rows (a decoding batch) with 4-bit weights:
 *   out[m, n] = sum_b s[g, b, n] * sum_{k in block b} x[m, k] q[g, k, n]
 * rows belonging to groups as in gl_gmm_fp8_fwd.
 *   x   bf16 [M, K];  w4, s in gl_quant_w4_128x1's format, q in -8..7 (a
 *       checkpoint's own scales will do);  group_sizes int32 [G] (device)
 *   out [M, N] bf16 or fp32 (out_dtype); rows at or past sum(group_sizes) are
 *       left as they are, or zeroed with GL_W4_ZERO_TAIL
 * Products are exact, sums fp32 (finite while those of |x q| over a block of 128
 * k stay below 2^134).  A non-finite x makes its row's outputs non-finite.
 * K % 128 == 0, N % 32 == 0, 1 <= G <= 1024, M <= 65536; x, w4, s, out and the
 * workspace 16-byte aligned.  The weights of a group are read once for every 8
 * rows of it: from about 16 rows a group on gl_gmm_fp8_fwd is the better choice.
 * workspace: gl_gmm_w4_workspace_bytes(M, K) bytes on the current device (0 for
 * an unsupported shape or M == 0), not used by another call in flight; what it
 * holds before does not matter, but for a captured call that ended with
 * GL_DEV_WAIT_TIMEOUT: clear it before that graph is replayed.  Negative sizes or
 * a sum past M set GL_DEV_BAD_GROUPS (out is then unspecified).
 */
size_t gl_gmm_w4_workspace_bytes(int64_t M, int64_t K);
int gl_gmm_w4_fwd(const void* x, const void* w4, const float* s, const int32_t* group_sizes, int64_t G,
                  int64_t M, int64_t K, int64_t N, void* out, int out_dtype, int flags, void* workspace,
                  size_t workspace_bytes, int* err_word, void* stream);

/* Largest M*K accepted by gl_gmm_fp8_act_fwd_noalloc (activation elements). */
#define GL_NOALLOC_MAX_ACT_ELEMS (16u * 1024u * 1024u)

/*
 * Grouped matmul forward from bf16 activations that allocates no device
 * memory.  No counterpart in the reference: it exists for callers that
 * cannot allocate device memory during a step (runtimes that plan every
 * buffer up front and forbid allocation while executing, FFI callers
 * without a device allocator).  It quantises lhs (1x128, as
 * gl_quant_act_1x128) into a fixed device scratch array owned by the
 * library (16 MiB of e4m3 plus 512 KiB of scales, created when the
 * library's device code loads on a GPU and held until exit) and runs
 * gl_gmm_fp8_fwd on it.
 *   lhs bf16 [M, K] with M * K <= GL_NOALLOC_MAX_ACT_ELEMS (else GL_EINVAL);
 *   b_q, b_s, group_sizes, out, out_dtype as gl_gmm_fp8_fwd.
 *   err_word: caller-owned device int for device-side error codes (invalid
 *   group_sizes, a wait that gave up).  Callers that need those errors must
 *   pass one: with NULL they go to the scratch array's own word, which every
 *   call clears first and which nothing reads back (gl_device_status(NULL)
 *   reads the library word, which this entry point never touches because
 *   that word is allocated memory).
 * All calls on a device share the scratch array and it keeps the last
 * call's contents; calls whose GPU work overlaps race on it.  The first call
 * on each device looks up the array's device address; make it before any
 * stream capture.
 */
int gl_gmm_fp8_act_fwd_noalloc(const void* lhs, const void* b_q, const float* b_s,
                               const int32_t* group_sizes, int64_t G, int64_t M,
                               int64_t K, int64_t N, void* out, int out_dtype,
                               int* err_word, void* stream);

/*
 * Synchronises `stream`, reads the device error word (the library word when
 * err_word is NULL) into *code and clears it.  Returns GL_OK or GL_ELAUNCH.
 */
int gl_device_status(int* err_word, void* stream, int* code);

/* Message of the last failing call on this host thread ("" if none). */
const char* gl_last_error(void);

/* Library version string. */
const char* gl_version(void);

#ifdef __cplusplus
}
#endif

#endif /* GLAUCIS_B200_H */
