/*
 * llamini_b200.h -- additive C entry points of the B200 library.
 *
 * Everything here is new: the reference (llamini.cpp) has no GPU, no batching
 * and no device-resident sessions, so none of these functions replaces a
 * reference symbol one-for-one. Each comment names the reference code whose
 * behaviour the function exposes or extends. All functions return 0 on success
 * and -1 on failure unless stated otherwise; the reason is kept in
 * llamini_last_error(). No function aborts the process.
 */
#ifndef LLAMINI_B200_H
#define LLAMINI_B200_H

#include "common.h"
#include "gguf.h"
#include "model.h"
#include "gpt2.h"
#include "kv_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- runtime --------------------------------------------------------------- */

/* Sticky description of the last failure ("" if none). The reference reports
 * errors only through -1 returns and stderr (gguf.h comments, main.c:472-477). */
const char* llamini_last_error(void);
void llamini_clear_error(void);

/* Number of visible CUDA devices (0 without a GPU; never fails). */
int llamini_device_count(void);

/* Select the CUDA device used by every later call of this process. Must be
 * called before the first model is loaded. Default: device 0, or the value of
 * the LLAMINI_DEVICE environment variable. */
int llamini_set_device(int device);

/* The library's CUDA stream (a cudaStream_t) on the current device, created on
 * first use; NULL without a device. Timing code records events on it. */
void* llamini_stream(void);

/* Release every device resource the library holds (weights, KV caches, graphs). */
void llamini_release(void);

/* ---- block decoders and GEMV on raw blocks (the gguf.c:409-594 and
 *      model.c:66-176 hot loops, exposed without a GGUF file) ------------------ */

/* Bytes taken by n_elems elements of ggml `type` (0 if the type is unsupported
 * or n_elems is not a multiple of its block size). */
u64 llamini_type_bytes(u32 type, u64 n_elems);

/* Decode n_elems elements of raw `type` blocks from host memory into host f32
 * out, on the GPU. Bit-identical to gguf.c:409-594. */
int llamini_dequant_host(u32 type, const void* blocks, u64 n_elems, f32* out);

/* One sample_token draw (generate.c:25-60) by the device sampler that the
 * sampled generate path uses: logits in host memory (vocab floats), temp > 0,
 * top_p, and u = rand() / (RAND_MAX + 1) as the reference computes it (the
 * caller draws it, so the host rand() stream is consumed in the reference's
 * order). Returns the token id, or 0xFFFFFFFF on error. */
u32 llamini_sample_host(const f32* logits, u32 vocab, f32 temp, f32 top_p, f32 u);

/* Same decode between device buffers, enqueued on llamini_stream(). */
int llamini_dequant_device(u32 type, const void* d_blocks, u64 n_elems, f32* d_out);

/* y[b][r] = sum_k W[r][k] * x[b][k] for b < batch, W given as raw `type` rows of
 * `cols` elements (cols a multiple of the block size). Host buffers; x is
 * batch x cols f32, y is batch x rows f32 (model.c:66-73 per column). */
int llamini_gemv_host(u32 type, const void* w, u32 rows, u32 cols,
                      const f32* x, u32 batch, f32* y);

/* Device-pointer form of llamini_gemv_host, enqueued on llamini_stream(). */
int llamini_gemv_device(u32 type, const void* d_w, u32 rows, u32 cols,
                        const f32* d_x, u32 batch, f32* d_y);

/* Decode attention for one query position over caller-owned DEVICE buffers,
 * with no device allocation. No counterpart in the reference: it computes what
 * causal_mha (model.c:217-260) computes after the cache already holds position
 * pos (the reference stores k/v first, model.c:222-224). d_q and d_out are
 * n_heads x head_dim f32; d_key/d_val are f32 caches laid out like KVCache
 * (row p = position p, n_heads_kv x head_dim) holding rows 0..pos. The work is
 * enqueued on `stream` (a cudaStream_t; NULL = the legacy default stream) of the
 * calling thread's current device.
 * For callers that may not allocate on their path (an engine whose page pool
 * already holds nearly all of HBM, a loop that cannot take cudaFree's implicit
 * device synchronisation): split partials and completion counters live in a
 * fixed 1 MiB (+1 KiB) array in the library's device memory. Limits: n_heads
 * <= 256, head_dim <= 256; larger requests fail with -1 and a message. The
 * counters start at zero and every call returns them to zero. The first call
 * on a device does the set-up (scratch address, kernel attribute) and should
 * come before any stream capture; it is kept for the life of the process, so
 * it does not survive a cudaDeviceReset of that device by the application.
 * Calls that overlap in time on one device (two streams, or unordered host
 * threads) share the scratch and race. */
int llamini_causal_mha_noalloc(const f32* d_q, const f32* d_key, const f32* d_val, f32* d_out,
                               u32 pos, u32 n_heads, u32 n_heads_kv, u32 head_dim, void* stream);

/* ---- 8-bit integer operators (no counterpart in the reference, whose products
 *      decode each weight to f32: model.c:66-176) ------------------------------
 *
 * A decoder layer's matrices as int8 x int8 products on the tensor cores: int8
 * weights with one scale for each output channel, activations with one scale
 * for each token. A row q[0..cols) with its scale stands for the values
 * q[i] * scale, where scale = max|y| / 127 and q = y * (127 / max|y|) rounded to
 * the nearest integer, ties to even (both quotients rounded to f32; the norm rounds
 * the factor once more, so that an element within 2^-16 of halfway may go the other
 * way, and its sums' order, with it their last bits, goes by the rows' length, number
 * and layout). A row of zeros has scale 0; a row that holds a NaN or an infinity has
 * scale NaN and q = 0.
 *
 * Every call takes DEVICE buffers of the calling thread's current device (others
 * are refused) and enqueues its work on `stream` (a cudaStream_t; NULL = the
 * legacy default stream). None allocates, keeps anything from call to call or
 * uses scratch, so calls may overlap in time and may be captured into graphs.
 * Matrices are row-major; a pitch ld_* counts elements from row to row and is at
 * least the row's length. What lies between a row's end and the next row's start
 * is not written, and its values do not matter. Pitches in multiples of 16 elements
 * from a 16-byte aligned base are what the fast kernels take; other ones work, slower. 1 to
 * 131071 columns; rows = 0 is a call without work. Outputs must not overlap
 * inputs, but for the sum of llamini_rms_norm_i8_device. */

/* Element types of activations: GGML_TYPE_F32, GGML_TYPE_F16 and */
#define LLAMINI_TYPE_BF16 30

/* Activations of llamini_glu_i8_device: ACT_SILU, ACT_GELU (model.h) and */
#define LLAMINI_ACT_NONE 2

/* int8 rows of raw GGUF blocks: the `cols` elements of each of `rows` rows,
 * decoded as by llamini_dequant_device (bit-identical to gguf.c:409-594), and the
 * row's scale. d_blocks holds whole rows back to back (2-byte aligned; F32 4-byte), d_q is rows x ld_q, d_scale
 * holds `rows` floats. Done once per matrix, when a model is loaded. */
int llamini_weights_i8_device(u32 type, const void* d_blocks, u32 rows, u32 cols,
                              i8* d_q, u64 ld_q, f32* d_scale, void* stream);

/* RMS norm of each row with the residual's addition, rounded to int8:
 * h = x + resid in f32 (x alone when d_resid is NULL), y = h / sqrt(mean(h^2) +
 * eps) * w (rms_norm, model.c:4-10), q and scale of y. x, resid and sum are of
 * `type`. d_sum (NULL: not stored) receives h rounded to `type`; it may be d_x or
 * d_resid, with that input's pitch, to update a residual stream in place. d_w
 * holds `cols` floats. A row whose sum of squares passes f32's range (finite values past
 * 1e19, say), or whose mean(h^2) + eps is below 2^-120, has scale NaN and q = 0. */
int llamini_rms_norm_i8_device(u32 type, const void* d_x, u64 ld_x, const void* d_resid, u64 ld_resid,
                               void* d_sum, u64 ld_sum, const f32* d_w, f32 eps, u32 rows, u32 cols,
                               i8* d_q, u64 ld_q, f32* d_scale, void* stream);

/* y = act(gate) * up, or act(gate) when d_up is NULL (ffn_glu, model.c:14-25;
 * with LLAMINI_ACT_NONE and no up, the rounding of plain rows to int8), q and
 * scale of y. act(x) is x / (1 + exp(-z)) in f32 (z = x for SiLU, 2 u for GELU's
 * 1 + tanh u), zero where 1 + exp(-z) passes f32's range (z below -88.7). gate and up are of `type` and may lie side by side in one buffer,
 * as one product of both matrices leaves them. */
int llamini_glu_i8_device(u32 type, const void* d_gate, u64 ld_gate, const void* d_up, u64 ld_up, u32 act,
                          u32 rows, u32 cols, i8* d_q, u64 ld_q, f32* d_scale, void* stream);

/* out[m][j] = (sum_k a[m][k] w[j][k]) * a_scale[m] * w_scale[j] (+ bias[j]) for
 * m < rows, j < n: the sum exact in 32-bit integers, the rest in f32, rounded to
 * out_type (F32, F16, BF16). d_bias may be NULL. a is rows x cols, w n x cols. An
 * output's bits do not depend on the other rows or channels of the call. */
int llamini_gemm_i8_device(const i8* d_a, u64 ld_a, const f32* d_a_scale, u32 rows,
                           const i8* d_w, u64 ld_w, const f32* d_w_scale, u32 n, u32 cols,
                           const f32* d_bias, u32 out_type, void* d_out, u64 ld_out, void* stream);

/* The longest that a product's kernel waits for its own copies and tensor-core
 * products before it gives up (its outputs are NaN then), for the calls that follow from
 * any thread: 2 s unless set, at most 60 s. With 0 such a kernel gives up without
 * waiting, which shows a caller's handling of llamini_i8_status without a fault
 * (products of one or two tokens, of up to eight where they take the same kernel, and
 * from rows that are not in 16-byte pitches have no waits to run out). */
int llamini_set_i8_wait_ns(u64 ns);

/* Waits for `stream`, then 0, or -1 when a bounded wait inside a product's kernel has
 * run out on the current device, on this stream or another, since the last call for
 * this stream (for its first: since the library was loaded). The outputs of such a
 * product are NaN; a call for one stream takes nothing away from another's. A
 * stream that is being captured is refused, and its capture goes on; so do the captures
 * of other streams. */
int llamini_i8_status(void* stream);

/* ---- device-resident decoding sessions (generate.c:122-167 without host
 *      round trips) --------------------------------------------------------- */

typedef struct llamini_session llamini_session;

/* Session for a loaded LLaMA-family model and its per-layer caches. The session
 * owns the device KV cache, the step graph and the token buffer; it is created
 * on first use by forward_step/generate_autoregressive as well, and this call
 * returns that same session. NULL on failure. */
llamini_session* llamini_llama_session(LLaMAModel* model, KVCache* caches);

/* Same for a GPT-2 model (gpt2.c:150-229). */
llamini_session* llamini_gpt2_session(GPT2Model* model, KVCache* caches);

/* Reset the session to position 0 with the given prompt (n_prompt >= 1). */
int llamini_session_begin(llamini_session* s, const u32* prompt, u32 n_prompt);

/* Enqueue n_steps forward passes without waiting. Step at position p embeds
 * token[p]; when p+1 >= n_prompt it also stores the greedy token as token[p+1].
 * Fails if the run would pass the cache capacity. */
int llamini_session_step(llamini_session* s, u32 n_steps);

/* Wait for queued steps, then copy token[0..n) to host out. Returns the number
 * of valid tokens (prompt + generated), or -1. */
int llamini_session_tokens(llamini_session* s, u32* out, u32 n);

/* Wait, then copy the logits of the most recent step (vocab_size floats). */
int llamini_session_logits(llamini_session* s, f32* out);

/* Current position (number of tokens already run through the stack). */
u32 llamini_session_pos(llamini_session* s);

/* How the session runs its steps: 2 = the dataflow decode kernel (one
 * cooperative launch for up to 64 steps; the default for LLaMA-family models
 * whose matrices are all Q4_K / Q6_K with K a multiple of 256 up to 6144),
 * 1 = the earlier persistent decode kernel (LLAMINI_DECODE_KERNEL=1 at session
 * creation, every matrix Q4_K, Q6_K, Q8_0 or Q4_0), 0 = one graph of per-op
 * kernels per step (every other model, or LLAMINI_DECODE_KERNEL=0); -1 = NULL. */
int llamini_session_kernel(llamini_session* s);

/* Algorithmic bytes one step reads: every weight matrix once, norms, biases and
 * one embedding row (the quantized sizes of gguf.c's block formats). */
u64 llamini_session_weight_bytes(llamini_session* s);

/* KV-cache bytes per cached position (all layers, K and V). */
u64 llamini_session_kv_bytes_per_pos(llamini_session* s);

/* Element type of the device KV cache of sessions created from now on:
 * 0 = f32 (default; the reference keeps an f32 cache, model.c:222-224, and the
 * f32 cache holds the 1e-3 parity bar), 1 = fp16 (half the cache traffic; on
 * the synthetic models its rounding moves logits by ~2e-3 relative L2). */
int llamini_set_kv_f16(int enable);

/* ---- batched decode (no counterpart in the reference, which decodes one
 *      sequence at a time: generate.c:122-167 run for each sequence) ---------- */

typedef struct llamini_batch llamini_batch;

/* A batch of up to max_batch (<= 64) independent sequences of at most max_seq
 * positions over a loaded model. Every weight matrix is read once per step for
 * the whole batch; the device KV cache holds max_batch x max_seq positions. The
 * matrices may be any of gguf.c's block formats or F16 with rows of a multiple
 * of 64 elements (256 for K-quants); NULL and a message otherwise.
 * Free it with llamini_batch_free before the model and its GGUF file. */
llamini_batch* llamini_llama_batch(LLaMAModel* model, u32 max_batch, u32 max_seq);
llamini_batch* llamini_gpt2_batch(GPT2Model* model, u32 max_batch, u32 max_seq);

/* Start n_seq sequences at position 0: prompts holds the n_seq prompts back to
 * back, prompt_lens their lengths (each >= 1). */
int llamini_batch_begin(llamini_batch* b, u32 n_seq, const u32* prompts, const u32* prompt_lens);

/* Enqueue n_steps positions of every sequence. At position p sequence s embeds
 * token[s][p]; once p + 1 is past its prompt its greedy token becomes
 * token[s][p + 1] -- per sequence exactly generate_autoregressive with temp 0
 * and no EOS (an EOS is for the caller to cut at). */
int llamini_batch_step(llamini_batch* b, u32 n_steps);

/* Wait, copy token[seq][0..n) to out; returns the number of valid tokens. */
int llamini_batch_tokens(llamini_batch* b, u32 seq, u32* out, u32 n);

/* Wait, copy the logits of sequence seq at the most recent step. */
int llamini_batch_logits(llamini_batch* b, u32 seq, f32* out);

u32 llamini_batch_pos(llamini_batch* b);
u64 llamini_batch_weight_bytes(llamini_batch* b);
void llamini_batch_free(llamini_batch* b);

/* Prompt positions whose logits nobody reads (generate_autoregressive's
 * prefill, llamini_session_step inside the prompt) run in chunks of 64
 * positions through the tcgen05 GEMM, with causal attention over the cache, when
 * every matrix takes the tensor-core path (one at a time otherwise): 1 = on (the
 * default), 0 = one position at a time, -1 = the default again
 * (LLAMINI_PREFILL=0 in the environment turns it off). The last prompt position
 * always runs through the decode step, which produces the logits. */
int llamini_set_prefill(int enable);

/* Whether this session's prompts have run through chunked prefill: 1 = yes (its
 * buffers are built), -1 = not available for this model (a format or shape the
 * tensor-core GEMM does not take, or a tensor-parallel group), 0 = not tried
 * yet; -2 = NULL. */
int llamini_session_prefill(llamini_session* s);

/* ---- tensor parallelism (no counterpart in the reference): LLaMA models split
 *      over the GPUs of one box, one process per GPU --------------------------- */

/* This process's 64-byte device-memory handle (a cudaIpcMemHandle_t) for the
 * allreduce buffer the other ranks read; pass every rank's to llamini_tp_join. */
int llamini_tp_handle(void* out64);

/* Join a group of `world` ranks as `rank`; handles = world handles of 64 bytes
 * in rank order. LLaMA sessions created afterwards hold this rank's shard:
 * heads [rank*H/world, (rank+1)*H/world) of q and o (o split by its columns),
 * the matching kv heads, and FFN columns split on 256-column boundaries (gate/up
 * rows, down columns); embeddings, norms and lm_head are whole, so every rank
 * computes the same logits. After the o projection and after ffn_down the
 * ranks' partial sums are added over NVLink (bounded waits; a rank that does not
 * arrive within 2 s sets the session's error). world = 1 leaves the group setting
 * at one rank. Prompt chunks (prefill) and batched sessions (LLaMA family, on
 * the tensor-core GEMM, at most 524288 / dim sequences) add their columns'
 * partial sums the same way, slice by slice. */
int llamini_tp_join(u32 rank, u32 world, const void* handles);
/* Leave the group (after the device has finished every step of the group's
 * sessions): unmaps the peers' buffers and clears this rank's buffer and
 * counters, so the process can join another group. Every rank of the group
 * leaves, and the ranks pass a host barrier before any of them joins again.
 * Sessions built in the group must not step afterwards. Returns 0 (also when
 * not in a group), -1 on a CUDA error. */
int llamini_tp_leave(void);
/* The shard a LLaMA session of rank `rank` in a group of `world` holds (the
 * plan llamini_tp_join's sessions use; no device needed): out[0..8) = {first
 * head, end head, first kv head, end kv head, first FFN column, end FFN column,
 * first o-proj column, end o-proj column}. FFN columns split on 256-column
 * super-block boundaries as evenly as they allow (first = 256 * floor(n_sb *
 * rank / world)). Returns 0, or -1 when the shapes do not split. */
int llamini_tp_plan(u32 world, u32 rank, u32 n_heads, u32 n_kv, u32 head_dim, u32 ffn, u32* out);
int llamini_tp_rank(void);
int llamini_tp_world(void);

/* Which GEMM a batch runs its matrices on: 1 = the tcgen05 tensor-core GEMM
 * (weights dequantised once per step into fp16 hi + lo, f32 accumulation in
 * tensor memory), 0 = the mma.sync GEMM; -1 = NULL. */
int llamini_batch_gemm_kind(llamini_batch* b);

/* GEMM for batched products (batches and the batch columns of llamini_gemv_*)
 * created or called from now on: 1 = tcgen05 (the default), 0 = mma.sync,
 * -1 = the default again (LLAMINI_BATCH_GEMM=mma in the environment selects
 * mma.sync). Shapes the tcgen05 GEMM does not take use mma.sync either way. */
int llamini_set_batch_gemm(int kind);

/* Per-layer residual stream of the most recent step: n_layers x dim floats,
 * captured when `enable` was set before the step ran. For parity tests. */
int llamini_session_trace(llamini_session* s, int enable);
int llamini_session_trace_read(llamini_session* s, f32* out);

#ifdef __cplusplus
}
#endif

#endif
