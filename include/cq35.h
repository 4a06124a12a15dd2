/*
 * cq35 — MI355X-native Qwen3.5/3.6 token loop behind a plain C ABI.
 *
 * The entry points replace the compiled catena artifact's session ABI that
 * hellas-ai/catena-models' Rust runtime binds (src/model.rs):
 *
 *   qwen3.init(capacity) -> state          src/model.rs:248-258,
 *                                          src/catena/state_init_moe.hex:2-13,
 *                                          src/catena/state_init_hybrid.hex:2-7
 *   qwen3(tokens, state, capacity, start,  src/model.rs:260-328,
 *         weights...) -> state, logits,    src/qwen/qwen35.rs:1466-1650
 *         token
 *   qwen3.copy-buffer(-16)(buffer, n)      src/model.rs:209-246,
 *                                          src/catena/session_copy.hex:131-135
 *   weights placed once in device memory   src/checkpoint.rs:197-231, 822-880
 *   weight ABI order                       src/spec.rs:443-712 (weight_specs)
 *
 * Conventions: every call returns 0 on success or a negative CQ35_E* code;
 * cq35_last_error() describes the last failure of the calling thread. No
 * signature carries framework types: only plain pointers, sizes and scalars.
 * One caller per session at a time; distinct sessions may be used from
 * distinct threads.
 */
#ifndef CQ35_H
#define CQ35_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CQ35_ABI_VERSION 3  /* 3: cq35_session_set_matrix_decode; 2: cq35_step_batch logits */

enum {
  CQ35_OK = 0,
  CQ35_EINVAL = -1,        /* malformed argument or configuration */
  CQ35_ERANGE = -2,        /* token id / position / capacity out of range */
  CQ35_EDEVICE = -3,       /* HIP runtime failure */
  CQ35_EUNSUPPORTED = -4,  /* path not provided by this build */
  CQ35_EPOISONED = -5      /* session state unusable after a failed step */
};

/* The fields of ModelConfig (src/spec.rs:33-62) the token loop reads.
 * moe != 0 selects ModelArchitecture::Qwen35Moe. */
typedef struct cq35_config {
  int32_t moe;
  int32_t vocab;
  int32_t hidden;
  int32_t intermediate;      /* dense FFN width, or per-expert width (MoE) */
  int32_t layers;
  int32_t q_heads;
  int32_t kv_heads;
  int32_t head_dim;
  int32_t rope_dim;
  float eps;
  float theta;
  int32_t experts;
  int32_t top_k;
  int32_t shared_intermediate;
  int32_t full_interval;
  int32_t key_heads;         /* linear_group_count */
  int32_t key_dim;           /* linear_state_size */
  int32_t value_heads;       /* linear_time_step_rank */
  int32_t value_dim;         /* linear_inner_size / linear_time_step_rank */
  int32_t tied;              /* output_weight_tied */
} cq35_config;

enum { CQ35_BF16 = 0, CQ35_F32 = 1 };

typedef struct cq35_tensor_info {
  int32_t dtype;      /* CQ35_BF16 or CQ35_F32 */
  int64_t rows;       /* leading dimensions folded: [E,I,H] -> rows=E*I, cols=H */
  int64_t cols;
  int64_t bytes;
} cq35_tensor_info;

typedef struct cq35_model cq35_model;
typedef struct cq35_session cq35_session;

const char* cq35_last_error(void);
int cq35_abi_version(void);

/* ModelConfig::validate (src/spec.rs:185-275) plus the limits of this build. */
int cq35_config_validate(const cq35_config* cfg);

/* weight_specs (src/spec.rs:443-712): tensor count and per-tensor shape. */
int cq35_weight_count(const cq35_config* cfg, int64_t* count);
int cq35_weight_info(const cq35_config* cfg, int64_t index, cq35_tensor_info* info);

/* Place the weights in device memory once (replacing the reference's
 * hipHostRegister zero-copy mapping, src/checkpoint.rs:916-986).
 * weights[i] points at tensor i in weight_specs order; on_device != 0 means
 * the pointers are already device allocations that the caller keeps alive
 * for the model's lifetime (they are borrowed, not copied). */
int cq35_model_create(const cq35_config* cfg, const void* const* weights, int on_device,
                      cq35_model** out);

/* Same, with weights produced on the device by the library's counter-based
 * synthetic generator: per tensor t and element i, SplitMix64 finaliser of
 * mix64(seed ^ mix64(t + 1)) + i * 0x9E3779B97F4A7C15, Irwin-Hall(4)
 * normals; BF16 matrices ~N(0, 0.02), norms 1 + N(0, 0.02), dt 1,
 * A = -(1 + 15u), conv N(0, 0.3), router N(0, 0.04), shared gate N(0, 0.02).
 * No reference counterpart: for benchmarks and parity tests without a
 * checkpoint. */
int cq35_model_create_synthetic(const cq35_config* cfg, uint64_t seed, cq35_model** out);

/* GGUF checkpoints (src/checkpoint.rs): `path` is one version-3 file, any
 * member of a standard shard set (<prefix>-NNNNN-of-MMMMM.gguf; every shard
 * is read) or a directory of .gguf files.
 * cq35_gguf_config: read_gguf_model_config (checkpoint.rs:376-404, 422-639)
 *   for the qwen35 / qwen35moe architectures (others: CQ35_EUNSUPPORTED);
 *   the output head is tied unless an output.weight tensor exists.
 * cq35_gguf_validate: validate_gguf_tensors (checkpoint.rs:406-414, 659-733,
 *   766-820): the tensor inventory equals weight_specs' GGUF names (tensors
 *   of next-token layers aside), each with its shape and dtype, inside its
 *   file, none overlapping. cfg, when given, must equal the metadata's.
 * cq35_model_load_gguf: Model::load_gguf (model.rs:43, 81-153): the above,
 *   then every tensor copied into HBM once (cq35_model_create).
 * cq35_gguf_tensor_name: the GGUF name of weight_specs entry `index`. */
int cq35_gguf_config(const char* path, cq35_config* out);
int cq35_gguf_validate(const char* path, const cq35_config* cfg);
int cq35_model_load_gguf(const char* path, cq35_model** out);
int cq35_gguf_tensor_name(const cq35_config* cfg, int64_t index, char* buf, int64_t len);
int cq35_model_free(cq35_model* model);
int cq35_model_config(const cq35_model* model, cq35_config* out);
/* Device bytes held by the model's weights. */
int cq35_model_weight_bytes(const cq35_model* model, int64_t* bytes);
/* Copy tensor `index` back to host memory (for checks). */
int cq35_model_read_weight(const cq35_model* model, int64_t index, void* dst, int64_t bytes);

/* qwen3.init: zero-initialised opaque state for `capacity` positions. */
int cq35_session_init(cq35_model* model, int64_t capacity, cq35_session** out);
int cq35_session_free(cq35_session* session);

/* qwen3: process tokens[0..n) at positions start..start+n (n == 1 is the
 * decode step), write the greedy next token and, when logits != NULL, the
 * final position's BF16 logits (vocab entries) to host memory.
 * `capacity` must equal the session's. A failure after work was enqueued
 * poisons the session (the reference drops its state on a failed exec,
 * src/model.rs:711-730). */
int cq35_step(cq35_session* session, const uint64_t* tokens, int64_t n, int64_t start,
              int64_t capacity, uint64_t* next_token, uint16_t* logits);

/* One decode step (one token each) for several independent sessions:
 * tokens[i] at position starts[i] of sessions[i], next token into
 * next_tokens[i] and, when logits != NULL, session i's BF16 logits into
 * logits[i * vocab ..]. Dense sessions of one model and capacity take one
 * weight-shared step (each layer's weights read once for all of them); each
 * session's result is then identical to its own cq35_step, unless every
 * session of the batch selects matrix-core decode
 * (cq35_session_set_matrix_decode), in which case the products run on MFMA
 * (hardware accumulation order: tolerance-level, like the matrix-core
 * prefill). Other sessions on the per-kernel path are launched back to back
 * on their own streams and then completed, so their kernels overlap on the
 * device; sessions on the persistent path step one at a time (each launch
 * needs every CU). All checks precede any work. If a step fails after work
 * was enqueued, every session of the batch is poisoned (some may have
 * advanced a position; none reports a token). No reference counterpart: the
 * reference steps sessions one after another (src/server/engine.rs:143-207);
 * this is the entry point for batch-16 serving. */
int cq35_step_batch(cq35_session* const* sessions, const uint64_t* tokens, const int64_t* starts,
                    int64_t count, uint64_t* next_tokens, uint16_t* logits);

/* A decode step (one token) that allocates nothing, for callers that cannot
 * allocate device memory: tight serving loops and harnesses that forbid
 * hipMalloc. No counterpart in the reference.
 * `state` is caller-owned device memory holding the BF16 session state of
 * `capacity` positions in the reference layout (cq35_session_state_bytes
 * with which = 0, e.g. copied from cq35_session_export_state); it is updated
 * in place exactly as cq35_step updates a session (same per-kernel decode
 * sequence, same results). `stream` is a hipStream_t (NULL: the default
 * stream); the call waits for it before returning the greedy token and, when
 * logits != NULL, the BF16 logits to host memory. Every other buffer comes
 * from one static device array of 16 MiB per device (held until the process
 * ends), which bounds the capacity: about 80K positions at the 35B-A3B shape;
 * larger capacities are rejected with CQ35_ERANGE before any work. Calls on
 * one device share that array: each holds a per-device lock from its first
 * launch until its stream has drained, so calls from several threads or
 * streams of one device run one after another. The call synchronises its
 * stream before returning, so it cannot run under HIP graph capture.
 * Decode attention splits above CQ35_SPLIT_KEYS_DEFAULT cached keys, as a
 * new session's does (there is no per-call threshold; at the capacities
 * this call accepts the split applies above 8192 positions). */
int cq35_step_static(const cq35_model* model, uint16_t* state, int64_t capacity, uint64_t token,
                     int64_t start, void* stream, uint64_t* next_token, uint16_t* logits);

/* qwen3.copy-buffer (session_copy.hex:131-135; src/model.rs:209-246): an
 * independent bitwise copy of a session's state and options. */
int cq35_session_copy(const cq35_session* src, cq35_session** out);

/* Canonical state for parity checks, in the reference layout
 * (state_layout.hex, decoder.hex:16-23, qwen35.hex:2-16):
 *   which = 0: BF16 cache [KV: layer, K|V, capacity, kv_heads*head_dim]
 *              [per layer: conv history 3*QKV, recurrent VH*VD*KD]
 *   which = 1: F32 DeltaNet shadow [layer, VH*VD*KD]
 *   which = 2: (MoE only, export only) int32 [layer, top_k]: the expert ids
 *              in rank order that the last call's final token selected at
 *              each layer (the reference keeps the current layer's ids in
 *              its workspace, state_layout.hex:53-87, written by
 *              qwen35_moe.hex:86-252)
 * `bytes` must equal cq35_session_state_bytes(session, which). */
int cq35_session_state_bytes(const cq35_session* session, int which, int64_t* bytes);
int cq35_session_export_state(const cq35_session* session, int which, void* dst, int64_t bytes);
int cq35_session_import_state(cq35_session* session, int which, const void* src, int64_t bytes);

/* Measurement hooks (no reference counterpart): time every launch of one
 * kernel class with start/stop events stamped by its dispatch packet on the
 * session stream (class ids: see cq35_kernel_class_name); -1 disables.
 * Results accumulate until read. Decode-step graph replay is suspended while
 * timing is on. */
int cq35_session_time_kernel(cq35_session* session, int kernel_class);
int cq35_session_kernel_time(cq35_session* session, double* total_ms, int64_t* launches);
const char* cq35_kernel_class_name(int kernel_class);
int cq35_kernel_class_count(void);
/* Phase stamps of the last persistent decode step, in a library built with
 * -DCQ35_PHASE_TRACE (otherwise CQ35_EUNSUPPORTED): `*slots` stamps per
 * block (s_memrealtime, 100 MHz) for each of the `*blocks` blocks of the
 * step; with dst != NULL, count must be blocks x slots. Slot meanings:
 * mega.h, phase trace. No reference counterpart (measurement only). */
int cq35_session_phase_trace(const cq35_session* session, uint64_t* dst, int64_t count, int64_t* slots,
                             int64_t* blocks);
/* Disable (0) or enable (1, default) hipGraph replay of the decode step. */
int cq35_session_set_graph(cq35_session* session, int enabled);

/* Decode steps (n == 1) of MoE models run as one persistent launch per token
 * by default, where the shape and capacity fit its limits; 0 selects the
 * per-kernel launch sequence, 1 the persistent kernel (CQ35_EUNSUPPORTED
 * when the session's shape is outside it). Same arithmetic either way. No
 * reference counterpart (the reference launches ~1,316 kernels per token). */
int cq35_session_set_persistent(cq35_session* session, int enabled);
int cq35_session_persistent(const cq35_session* session, int* enabled);

/* Split-K decode attention for long contexts. Over more than `keys` cached
 * keys (default CQ35_SPLIT_KEYS_DEFAULT; 0: never) the T tiles (8 keys) of
 * each query head's online softmax form at most 128 ranges of ceil(T / 128)
 * tiles, each the reference's recurrence over its own tiles from scratch,
 * merged in ascending range order (M = max m_r, w_r = exp(m_r - M),
 * den = 0 + d_0 w_0 + d_1 w_1 + ..., likewise each channel). The reference
 * runs one sequential chain over all tiles (qwen35_online.hex:272-331); the
 * split changes rounding only (tolerance-level), and at or below the
 * threshold the result is the reference's bit for bit. Both decode paths use
 * the same ranges, which depend on the key count alone. */
#define CQ35_SPLIT_KEYS_DEFAULT 8192
int cq35_session_set_attention_split(cq35_session* session, int64_t keys);
int cq35_session_attention_split(const cq35_session* session, int64_t* keys);

/* Matrix-core prefill: components of multi-token calls run on MFMA, whose
 * F32 accumulation order is the hardware's, so results match the exact path
 * to accumulation rounding rather than bit for bit. Replaces the reference's
 * InferenceOptions::wmma_prefill with CATENA_WMMA_COMPONENTS (catena.rs:12-26,
 * qwen35.rs:467-541; default off in its library API, as here). Bit 0: the
 * dense projections (attention, DeltaNet and output projections, dense FFN);
 * bit 1: the MoE expert projections (grouped routed experts and the shared
 * expert); bit 2: the full-attention layers' attention over the prompt rows
 * (scores and context on MFMA with the reference's BF16 score, probability
 * and context rounding, qwen35_wmma_attention.hex; head_dim 64, 128 or 256,
 * other head dims keep the exact kernels). 0 keeps the exact SIMT path. Calls
 * with a component run in chunks of 2048 tokens, others of 1024 (1024 and 256
 * where device memory is short; the chunk changes no result), in buffers lent
 * for the length of the call: calls that run at the same time each hold
 * theirs, sessions between calls none. Decode steps (cq35_step with n == 1, and
 * cq35_step_batch) are unaffected, as the reference's option affects prefill
 * only. */
#define CQ35_MATRIX_PROJECTIONS 1
#define CQ35_MATRIX_EXPERTS 2
#define CQ35_MATRIX_ATTENTION 4
int cq35_session_set_matrix_prefill(cq35_session* session, int components);
int cq35_session_matrix_prefill(const cq35_session* session, int* components);

/* One-pass attention of multi-token calls (no reference counterpart): 1 runs
 * the attention component (CQ35_MATRIX_ATTENTION, which has to be selected for
 * it to matter) as cq35_paged_attention over the session's cache: a running
 * maximum and sum instead of two passes over the keys, scores and probabilities
 * kept in F32 where the reference's matrix-core path rounds them to BF16 (the
 * unnormalised weights enter the second product as BF16), keys split over the
 * device where a call has few rows: how a prompt is divided into calls changes
 * its rounding, how much device memory is free does not.
 * Tolerance-level, as the component is; 0 (the default) keeps the reference's
 * rounding points. head_dim 64, 128 or 256; sessions of more than 2^22 positions
 * keep the two passes. Prompt buffers hold up to 135 MB more. Copied by
 * cq35_session_copy. */
int cq35_session_set_online_attention(cq35_session* session, int enabled);
int cq35_session_online_attention(const cq35_session* session, int* enabled);

/* Matrix-core batched decode (no reference counterpart): 1 lets the
 * weight-shared step of cq35_step_batch run its products on MFMA (hardware
 * accumulation order, tolerance-level) for a batch in which EVERY session has
 * this option set; a batch with any session at 0 (the default) takes the
 * exact products, so each session's tokens are then identical to its own
 * cq35_step. Single-session steps are unaffected. Copied by
 * cq35_session_copy. */
int cq35_session_set_matrix_decode(cq35_session* session, int enabled);
int cq35_session_matrix_decode(const cq35_session* session, int* enabled);

/* Host-side builds of the device numerics (same source), for CPU checks. */
float cq35_numeric_exp(float x);
float cq35_numeric_sqrt(float x);
float cq35_numeric_softplus(float x);
void cq35_numeric_sincos(float angle, float* sine, float* cosine);
/* Device evaluation of the same numerics over an array (op 0 exp, 1 silu,
 * 2 sigmoid, 3 softplus, 4 sqrt, 5 sin, 6 cos, 7 the F32 -> BF16 rounding
 * widened back to F32); host in/out arrays. */
int cq35_device_numeric(int op, const float* input, float* output, int64_t count);
/* Device split-pair GEMV with tree width W (32, 64 or 256) over a row-major
 * BF16 matrix: out[r] = bf16(tree_W(x . w_r)). Host arrays. */
int cq35_device_gemv(const uint16_t* x, const uint16_t* w, int64_t rows, int64_t cols,
                     int width, uint16_t* out);
/* Device matrix-core product of the prefill projections over host arrays,
 * x [n][cols], w and w2 [rows][cols], res [n][rows], cols a multiple of 16:
 * out[t][r] = epilogue(sum_k x[t][k] w[r][k]) in the MFMA accumulation order,
 * mode 0 bf16(sum), 1 bf16(sum) (+) res, 2 bf16(silu(bf16 sum)) (x)
 * bf16(sum over w2). kernel 0: direct fragment loads; 1: the LDS-staged
 * tiles the prefill runs (the same order, so the same bits). */
int cq35_device_matrix_gemm(const uint16_t* x, const uint16_t* w, const uint16_t* w2,
                            const uint16_t* res, int64_t n, int64_t rows, int64_t cols, int mode,
                            int kernel, uint16_t* out);
/* Device exact product of the prompt projections (the reference's batched
 * order, one accumulator per lane of 256) over host arrays laid out as above,
 * cols a multiple of 8, the same epilogues. kernel 0: the vector kernel; 1:
 * the kernels a prompt of n tokens runs (eight tokens or more of widths in
 * whole 128-byte lines: the F32 matrix cores and the recomputation of what
 * they would round differently). The same bits. */
int cq35_device_exact_gemm(const uint16_t* x, const uint16_t* w, const uint16_t* w2,
                           const uint16_t* res, int64_t n, int64_t rows, int64_t cols, int mode,
                           int kernel, uint16_t* out);
/* Device matrix-core attention of the prompt path (CQ35_MATRIX_ATTENTION's
 * kernel) over host arrays: n query rows at positions start .. start + n - 1
 * against keys 0 .. start + n - 1. q and gate [n][heads][head_dim] (q
 * normalised and rotated), k and v [start + n][kv_heads][head_dim], out
 * [n][heads][head_dim] = bf16(bf16(sum_j p_j v_j) * sigmoid(gate)) with
 * p_j = bf16(exp(s_j - max) / den) and s_j = bf16(q . k_j / sqrt(head_dim))
 * over the keys j at or before the row's position, the products on MFMA.
 * head_dim 64, 128 or 256; heads a multiple of kv_heads. */
int cq35_device_matrix_attention(const uint16_t* q, const uint16_t* gate, const uint16_t* k,
                                 const uint16_t* v, int64_t n, int64_t start, int heads, int kv_heads,
                                 int head_dim, uint16_t* out);

/* ---------------------------------------------------------- paged KV cache
 * Operators over device memory for callers that serve many requests from one
 * pool of cache pages beside their own projections: pages and slots of a
 * round (cq35_page_plan), head norm + rotation + append (cq35_paged_prepare)
 * and attention (cq35_paged_attention). No reference counterpart (its cache
 * is one contiguous block per session, state_layout.hex:26-27).
 *
 * Every pointer is device memory (of one device, which need not be the
 * calling thread's current one) unless its comment says host. A call checks
 * its arguments, enqueues its kernels on `stream` (a hipStream_t of that
 * device; NULL: its default stream) and returns; it allocates and waits for
 * nothing, so it may be captured into a graph. Buffers stay valid until the
 * work has run. Numbers in device memory (lengths, tables, slots) are read by
 * the kernels, which never leave the buffers whatever they hold: what a wrong
 * number does is said with each operator. */

/* Keys and values of `pages` pages of `page_size` rows (a power of two, 16 to
 * 65536), BF16. Row o of page p, head h starts at p * page_stride +
 * o * row_stride + h * head_stride elements of `keys` and `values` (both laid
 * out alike) and holds head_dim (64, 128 or 256) elements. Strides are
 * multiples of 8, the bases 16-byte addresses; pages, rows and heads may
 * follow each other in any order but not overlap. pages * page_size is below
 * 2^31. */
typedef struct cq35_paged_cache {
  void* keys;
  void* values;
  int64_t pages;
  int32_t page_size;
  int32_t kv_heads;
  int32_t head_dim;
  int64_t page_stride;
  int64_t row_stride;
  int64_t head_stride;
} cq35_paged_cache;

/* Rows of heads, BF16: head h of row t starts at t * row_stride +
 * h * head_stride elements. Strides are multiples of 8 (0 repeats a row of an
 * input), the base a 16-byte address. */
typedef struct cq35_heads {
  void* data;
  int64_t row_stride;
  int64_t head_stride;
} cq35_heads;

/* The pages, positions and slots of a round: request r holds cached[r] tokens
 * and is to hold lengths[r]. A longer one gets lengths[r] - cached[r] rows and
 * the pages they need; a shorter one (0: finished) gives back the pages it no
 * longer needs. Tables hold `width` page numbers, row r at r * table_stride;
 * those of the first ceil(cached[r] / page_size) entries are read.
 * `free_pages` is a stack of `pages` entries, the first *free_count of them
 * free pages. Pages given back are pushed first, in request and table order,
 * then the needed ones are popped in request and table order.
 * Written: the tables' new entries; free_pages; row_start[requests + 1] (the
 * exclusive sums of the requests' rows); positions and slots of `rows` rows (a
 * row's slot is page * page_size + position % page_size; rows behind the last
 * request's get position 0 and slot -1, also a row of an entry outside the
 * pages); *free_left (the count after; not free_count itself); status[2]: 0, or
 * 1 pages are missing (status[1] of them), 2 `rows` is too small (by
 * status[1]), 3 a length is negative or longer than a table, 4 the stack's
 * count is negative or, with the pages given back, above `pages`. Unless
 * status[0] is 0 the tables and the stack are left as they were, row_start is 0
 * and every slot -1: later operators of the round then do nothing. Outputs
 * overlap neither each other nor inputs, the tables and free_pages apart.
 * requests: 1 to 8192. With the same free_count the call can be repeated with
 * the same results. */
int cq35_page_plan(int32_t* table, int64_t table_stride, int64_t requests, int64_t width,
                   const int32_t* cached, const int32_t* lengths, int32_t* free_pages, int64_t pages,
                   const int32_t* free_count, int32_t page_size, int64_t rows, int32_t* row_start,
                   int32_t* positions, int32_t* slots, int32_t* free_left, int32_t* status,
                   void* stream);

/* Head norm, rotation and append of `rows` rows of projections: queries
 * q_out = rotate(norm(q, q_weight)), keys rotate(norm(k, k_weight)) into cache
 * row slots[t], values copied there. norm(x, w) = x w / sqrt(mean(x^2) + eps)
 * over a head's channels (w: F32, head_dim entries at a 16-byte address);
 * rotate turns channels i and i + rope_dim / 2 by position * inv_freq[i]
 * (inv_freq: F32, rope_dim / 2 entries; rope_dim a multiple of 16), the
 * position that of axis pair_axis[i] (host, rope_dim / 2 entries below `axes`;
 * NULL with one axis): positions[axis * position_stride + t], up to 4 axes
 * (time, height and width of images; a stride of 0 repeats one row of positions
 * on every axis, others are at least `rows`). F32 inside, the angle modulo a
 * turn in 64 bits, each result rounded to BF16 once; a head whose mean square
 * passes F32's range gives zeros. q_out may be q itself, laid out
 * alike. A row whose slot is negative or past the cache is left alone: neither
 * its query nor the cache is written. Slots of one call differ; of two equal
 * ones either row may end up in the cache, piece by piece. Up to 2^26 rows. */
int cq35_paged_prepare(const cq35_paged_cache* cache, const cq35_heads* q, const cq35_heads* k,
                       const cq35_heads* v, int64_t rows, int32_t q_heads, const float* q_weight,
                       const float* k_weight, float eps, const float* inv_freq, int32_t rope_dim,
                       const int32_t* positions, int64_t position_stride, int32_t axes,
                       const uint8_t* pair_axis, const int32_t* slots, const cq35_heads* q_out,
                       void* stream);

/* Attention of new tokens over the cache: rows row_start[r] up to
 * row_start[r + 1] of q are the last tokens of request r, which holds
 * lengths[r] tokens (theirs included) in the pages of table row r (`width`
 * entries at r * table_stride). Row i of n is at position p = lengths[r] - n
 * + i and sees the keys at positions 0 .. p:
 *   out = sum_j softmax_j(scale q . k_j) v_j, times sigmoid(gate) where gate
 * is not NULL; query head h reads key/value head h * kv_heads / q_heads.
 * Products on the matrix cores with F32 sums; the weights e^(s - max) enter
 * the second product as BF16 (off by at most 2^-8 each, as the values they
 * meet), the sums and the running maximum stay F32, the result is rounded to
 * BF16 once. The same call gives the same bits.
 * A row that sees no key (p < 0), or none with a score above -inf, gets zeros,
 * whatever its values and its gate.
 * Keys in pages whose number is outside the cache are not seen; lengths are
 * cut to what the table holds (at most 2^30 keys). Rows outside every request
 * are left alone. row_start ascends from 0 or more: where it does not, rows of a
 * request that overlaps another's hold either's results or are left alone, as are
 * those of later requests; rows past `rows` are not read or written. Up to 8192 requests; rows * q_heads below about 2^27. out may be
 * q itself, laid out alike; it overlaps no other operand.
 * max_rows and max_keys are what the caller knows of the most rows and keys of
 * any request, 0 for nothing: they steer how the work is cut and the launches
 * spared, results hold whatever they say.
 * workspace: cq35_paged_attention_workspace bytes (of the same arguments) at
 * a 16-byte address, used during the call's work only and by no other work at
 * that time; NULL where 0 bytes are needed. */
int cq35_paged_attention_workspace(int64_t rows, int64_t requests, int32_t q_heads, int32_t kv_heads,
                                   int32_t head_dim, int64_t max_rows, int64_t max_keys,
                                   int64_t* bytes);
int cq35_paged_attention(const cq35_paged_cache* cache, const cq35_heads* q, const cq35_heads* gate,
                         const cq35_heads* out, int64_t rows, int32_t q_heads, const int32_t* table,
                         int64_t table_stride, int64_t requests, int64_t width,
                         const int32_t* row_start, const int32_t* lengths, float scale,
                         int64_t max_rows, int64_t max_keys, void* workspace,
                         int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
