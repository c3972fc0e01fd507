/*
 * promptboot_b200 -- C ABI of the B200 (sm_100a) decode hot path.
 *
 * Drop-in boundary for promptboot-core's model-forward and sampler entry points
 * (sulewicz/promptboot).  Every call returns a u32 status (0 = OK) and reports
 * failures through the 48-byte pb_error, whose layout and numbering are the
 * reference's InferenceError (crates/promptboot-core/src/inference.rs:155-264).
 * Floats never cross this ABI as floats: logits are binary32 bit patterns in
 * uint32_t, as in the reference (fp32_sse2.rs:1-6).  No C++ or torch types
 * appear here; pointers are host pointers unless the name says _device.
 *
 * Threading: a pb_engine is single-owner (like the reference's &mut engine);
 * use one engine per GPU and one host thread per engine.
 */
#ifndef PROMPTBOOT_B200_H
#define PROMPTBOOT_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define PB_API __attribute__((visibility("default")))
#else
#define PB_API
#endif

#define PB_ABI_VERSION 1u
#define PB_VOCAB 151936u
#define PB_CONTEXT_LIMIT 32768u
#define PB_MODEL_BYTES 426762944ull
#define PB_SEEN_BYTES 18992u

/* InferenceStatus (inference.rs:155-169) */
enum {
    PB_OK = 0, PB_STATE = 1, PB_CONTEXT = 2, PB_TOKEN_ID = 3, PB_CAPACITY = 4,
    PB_ALIGNMENT = 5, PB_NONFINITE_INPUT = 6, PB_NONFINITE_OUTPUT = 7, PB_MODEL = 8,
    PB_ARITHMETIC = 9, PB_FAULTED = 10,
    PB_DEVICE = 100 /* CUDA runtime failure; no reference counterpart */
};

/* InferenceState (inference.rs:217-224) */
enum { PB_STATE_RESET = 0, PB_STATE_READY = 1, PB_STATE_EOS = 2, PB_STATE_FAULTED = 3 };

/* pb_model_open flags: the synthetic images used here carry zeroed tokenizer
 * sections, so only the layout (header, sections, tensor directory) is checked. */
enum { PB_MODEL_LAYOUT_ONLY = 1u };

/* InferenceError (inference.rs:226-238), 48 bytes */
typedef struct pb_error {
    uint32_t status, domain, layer, position, tensor_id, reserved;
    uint64_t needed, available, detail; /* detail = (field_kind << 32) | sub */
} pb_error;

/* InferenceStep (inference.rs:266-273), 16 bytes */
typedef struct pb_step {
    uint32_t position, selected_token, selected_logit_bits, eos;
} pb_step;

/* ArenaUsage (arena.rs) and InferenceUsage (inference.rs:275-285), 136 bytes */
typedef struct pb_arena_usage {
    uint64_t capacity, requested, committed, current, high_water;
} pb_arena_usage;
typedef struct pb_usage {
    pb_arena_usage weights, kv, scratch;
    uint32_t position, context_limit, generation_reserve, state;
} pb_usage;

/* SamplingState (inference.rs:772-799), 16 bytes */
typedef struct pb_sampling_state { uint64_t state, draws; } pb_sampling_state;

/* TopLogit (inference.rs:759-770), 8 bytes */
typedef struct pb_top_logit { uint32_t token, logit_bits; } pb_top_logit;

/* ModelError (model.rs:113-124), 48 bytes */
typedef struct pb_model_error {
    uint32_t status, domain, index, reserved;
    uint64_t offset, needed, available, detail;
} pb_model_error;

typedef struct pb_model pb_model;
typedef struct pb_engine pb_engine;

PB_API uint32_t pb_abi_version(void);
/* Text of the last CUDA/runtime failure seen on this thread ("" when none). */
PB_API const char *pb_last_error_string(void);

/* ------------------------------------------------------------------ model
 * Replaces ModelView::open_authenticated (model.rs:371-629) + tensor/tensor_for
 * (model.rs:652-720).  Validates the PBTQW25 v1 layout, then uploads section 7
 * (tensor data) to `device` unchanged, in PBTQW25 byte order. */
PB_API uint32_t pb_model_open(const uint8_t *bytes, uint64_t len, uint32_t flags, int device,
                       pb_model **out, pb_model_error *err);
PB_API void pb_model_close(pb_model *model);
/* Device pointer of tensor `id` (model.rs:652) or NULL. */
PB_API const void *pb_model_tensor_device(const pb_model *model, uint32_t id);

/* ----------------------------------------------------------------- engine
 * Replaces InferenceEngine (inference.rs:967-1371).  One engine owns
 * `max_seqs` independent sequences ("slots"), each with its own KV cache of
 * `max_context` positions (<= 32768; the reference's fixed KV is 32768) in the
 * reference's tiled layout, its own state machine and retained prefix. */
PB_API uint32_t pb_engine_create(pb_model *model, uint32_t max_seqs, uint32_t max_context,
                          pb_engine **out, pb_error *err);
PB_API void pb_engine_destroy(pb_engine *engine);

/* inference.rs:1026 prefill / :1044 prefill_with_prefix / :1095 append_prefill.
 * `logits` (optional) receives the 151936 binary32 words of the last token. */
PB_API uint32_t pb_engine_prefill(pb_engine *engine, uint32_t seq, const uint32_t *tokens, uint32_t n,
                           uint32_t generation_reserve, uint32_t *logits, pb_step *step,
                           pb_error *err);
PB_API uint32_t pb_engine_prefill_with_prefix(pb_engine *engine, uint32_t seq, const uint32_t *tokens,
                                       uint32_t n, uint32_t prefix_tokens,
                                       uint32_t generation_reserve, uint32_t *logits,
                                       pb_step *step, pb_error *err);
PB_API uint32_t pb_engine_append_prefill(pb_engine *engine, uint32_t seq, const uint32_t *tokens,
                                  uint32_t n, uint32_t generation_reserve, uint32_t *logits,
                                  pb_step *step, pb_error *err);
/* inference.rs:1205 decode (token must equal the last greedy id) / :1213 decode_selected */
PB_API uint32_t pb_engine_decode(pb_engine *engine, uint32_t seq, uint32_t token, uint32_t *logits,
                          pb_step *step, pb_error *err);
PB_API uint32_t pb_engine_decode_selected(pb_engine *engine, uint32_t seq, uint32_t token,
                                   uint32_t *logits, pb_step *step, pb_error *err);
/* inference.rs:1307 reset / :1315 reset_to_prefix / :1337 usage / :1369 position */
PB_API uint32_t pb_engine_reset(pb_engine *engine, uint32_t seq);
PB_API uint32_t pb_engine_reset_to_prefix(pb_engine *engine, uint32_t seq, uint32_t *prefix_out);
PB_API uint32_t pb_engine_usage(pb_engine *engine, uint32_t seq, pb_usage *out);
PB_API uint32_t pb_engine_position(pb_engine *engine, uint32_t seq);

/* KV snapshot access (no counterpart in the reference, whose KV is a caller-
 * owned byte slice: InferenceEngine::build, inference.rs:977-1011).
 * pb_engine_kv_device returns the device address of slot `seq`'s KV region,
 * *words binary32 words = max_context * 6144, in the reference's tiled layout
 * (inference.rs:2035-2052) with the slot's capacity C in place of 32768:
 * K at layer*4C*64 + ((h*C/4 + p/4)*64 + c)*4 + p%4, V at layer*4C*64 + 2C*64 +
 * (h*C + p)*64 + c.  Reads and writes through it are the caller's, ordered
 * against the engine by synchronizing pb_engine_stream.
 * pb_engine_restore makes a RESET slot hold `tokens` (n < context limit) whose
 * KV of positions [0, n) the caller has written there (a saved snapshot):
 * prefill's prechecks (inference.rs:1109-1191) on tokens and reserve, then the
 * slot is READY at position n with history = tokens and no greedy id, so the
 * next call is decode_selected (decode reports the selected-token state error). */
PB_API void *pb_engine_kv_device(pb_engine *engine, uint32_t seq, uint64_t *words);
PB_API uint32_t pb_engine_restore(pb_engine *engine, uint32_t seq, const uint32_t *tokens, uint32_t n,
                                  uint32_t generation_reserve, pb_error *err);

/* Batched forms: one forward step over n distinct sequences at their own
 * positions (a sequence listed twice: PB_CAPACITY).  prefill_batch runs `len`
 * prompt tokens per sequence (tokens is [n][len]; positions but the last as
 * batched (sequence, position) rows, results as the token-serial reference);
 * decode_batch evaluates tokens[i] for seqs[i] (require_greedy = 1 is decode, 0
 * is decode_selected).  Per-sequence results land in steps[i]/errs[i]; the call
 * returns PB_OK when every sequence succeeded, else the first failing status.
 * Logits stay on the device (row i = seqs[i]); see pb_engine_logits. */
PB_API uint32_t pb_engine_prefill_batch(pb_engine *engine, uint32_t n, const uint32_t *seqs,
                                 const uint32_t *tokens, uint32_t len,
                                 uint32_t generation_reserve, pb_step *steps, pb_error *errs);
PB_API uint32_t pb_engine_decode_batch(pb_engine *engine, uint32_t n, const uint32_t *seqs,
                                const uint32_t *tokens, uint32_t require_greedy,
                                pb_step *steps, pb_error *errs);
/* Copies the logits row of batch row `row` of the last step to host. */
PB_API uint32_t pb_engine_logits(pb_engine *engine, uint32_t row, uint32_t *logits);
/* sample_token_with_repetition (inference.rs:919-965) on batch rows 0..n-1 of the
 * last step, history = every token seqs[i] has evaluated; states are host
 * SamplingStates updated in place; ids[i] = sampled token. */
PB_API uint32_t pb_engine_sample(pb_engine *engine, uint32_t n, const uint32_t *seqs,
                          pb_sampling_state *states, uint32_t *ids, pb_error *errs);
/* Device-resident generation (benchmark mode: fixed length, EOS not honoured):
 * `steps` times { sample the current logits rows with repetition history, then
 * decode_selected(sampled) }, all on the GPU.  Requires every seq READY/EOS with
 * logits from its last step in batch row i.  out_tokens (optional, host) is
 * [steps][n]. */
PB_API uint32_t pb_engine_generate(pb_engine *engine, uint32_t n, const uint32_t *seqs,
                            pb_sampling_state *states, uint32_t steps, uint32_t *out_tokens,
                            pb_error *errs);

/* Engine instrumentation (no reference counterpart): the CUDA stream every
 * engine kernel runs on, the number of kernels launched so far, and optional
 * CUDA-event timing of selected kernel classes (bit i of class_mask = class i
 * below) accumulated on that stream; pb_engine_profile also resets the sums. */
enum {
    PB_KC_EMBED = 0, PB_KC_NORM = 1, PB_KC_GEMV = 2, PB_KC_ROPE_KV = 3, PB_KC_ATTENTION = 4,
    PB_KC_QUANT = 5, PB_KC_SWIGLU = 6, PB_KC_LM_HEAD = 7, PB_KC_ARGMAX = 8, PB_KC_SAMPLER = 9
};
PB_API void *pb_engine_stream(pb_engine *engine);
PB_API uint64_t pb_engine_launch_count(pb_engine *engine);
PB_API uint32_t pb_engine_profile(pb_engine *engine, uint32_t class_mask);
PB_API uint32_t pb_engine_profile_read(pb_engine *engine, double *ms16, uint64_t *launches16);

/* ---------------------------------------------------------------- sampler
 * Host-buffer forms of the reference's sampler entry points, executed on the
 * GPU (inference.rs:814-965).  Error fields match the reference. */
PB_API void pb_sampling_state_init(pb_sampling_state *state, uint64_t seed);
PB_API uint32_t pb_sample_token(const uint32_t *logits, uint64_t len, pb_sampling_state *state,
                         uint32_t *out, pb_error *err);
PB_API uint32_t pb_sample_token_with_repetition(uint32_t *logits, uint64_t len, const uint32_t *tokens,
                                         uint64_t count, uint8_t *seen, uint64_t seen_len,
                                         pb_sampling_state *state, uint32_t *out, pb_error *err);
PB_API uint32_t pb_greedy_token(const uint32_t *logits, uint64_t len, uint32_t *out, pb_error *err);
PB_API uint32_t pb_top_logits_8(const uint32_t *logits, uint64_t len, pb_top_logit *out8, pb_error *err);

/* Device batch sampler: rows of binary32 logits (row stride ld words) mutated in
 * place by the penalty; history for row r is history[offsets[r] .. +lengths[r]];
 * states [rows] updated; out [rows] receives {status, index, value, selected}
 * (status 0 ok, 3 TOKEN_ID at history index/value, 7 NONFINITE_OUTPUT at
 * logit index/bits).  Asynchronous on `stream` (a cudaStream_t, NULL = default). */
PB_API uint32_t pb_sample_batch_device(uint32_t *logits_device, uint64_t ld, uint32_t rows,
                                const uint32_t *history_device, const uint64_t *offsets_device,
                                const uint32_t *lengths_device,
                                pb_sampling_state *states_device, uint32_t *out_device,
                                void *stream);

/* --------------------------------------------------------- kernel operators
 * Device-pointer operators behind the engine, for tests and operator sweeps.
 * All are asynchronous on `stream`. */
/* y[b][r] = Q4_0 (wtype 2) or Q8_0 (wtype 3) weights [rows][cols] times the
 * Q8_0-quantized x[b] (fp32_sse2.rs:945-983, 1217-1281); x is f32 [batch][cols].
 * Scratch: the quantized x; allocated per call. */
PB_API uint32_t pb_qmatvec_device(uint32_t wtype, const uint8_t *w_device, uint32_t rows, uint32_t cols,
                           const float *x_device, uint32_t batch, float *y_device, void *stream);
/* The same operator without any device allocation (no counterpart in the
 * reference): for callers that cannot allocate device memory on this path,
 * e.g. hosts that own the GPU's memory budget through their own allocator,
 * latency-critical loops, or fixed-arena integrations like promptboot's own
 * firmware runtime.  Its scratch is one file-scope device array of 192 KiB
 * held by each GPU that loads the library; batch is limited to 32 rows and
 * cols to 4864 (PB_CAPACITY otherwise, see pb_last_error_string).  The first
 * call on a device sets it up and should come before any stream capture; all
 * calls share the array, so calls whose kernels overlap on the GPU (queued on
 * different streams, from any thread) race; calls queued on one stream are
 * ordered by it.  Unlike pb_qmatvec_device it does not wait: it returns once
 * the work is queued on `stream`, and y is ready when that stream has reached
 * it.  Non-finite outputs are not reported (y holds them as computed).  The
 * array's device address is looked up once per device for the process, so the
 * call must not be used after a cudaDeviceReset of that device. */
PB_API uint32_t pb_qmatvec_device_noalloc(uint32_t wtype, const uint8_t *w_device, uint32_t rows,
                                          uint32_t cols, const float *x_device, uint32_t batch,
                                          float *y_device, void *stream);
/* y[b] = model tensor `tensor_id` (a layer's q/k/v/o/gate/up/down matrix, the
 * Q8_0 output head, id 290, or the Q4_0 token embedding, id 0, as a tied
 * 896 -> 151936 head) times the Q8_0-quantized x[b], x f32 [batch][cols]:
 * the engine's own matvec (the tensor-core path on the model's tile image from
 * 9 rows, the CUDA-core path below).  Asynchronous on `stream`, no per-call
 * allocation once the model's scratch has grown to the batch (batch <= 256;
 * tensor 0's tile image is built on its first call from 9 rows);
 * pb_model_matvec_status synchronizes `stream` and reports a pipeline timeout of
 * any earlier call (PB_DEVICE) once.  Replaces the row loop of
 * inference_q4_matvec_rows_prepared / inference_q8_matvec_rows_prepared
 * (fp32_sse2.rs:1217-1281) over ModelView::tensor (model.rs:652). */
PB_API uint32_t pb_model_matvec_device(pb_model *model, uint32_t tensor_id, const float *x_device,
                                       uint32_t batch, float *y_device, void *stream);
PB_API uint32_t pb_model_matvec_status(pb_model *model, void *stream);
/* Q8_0 staging in the reference's 34-byte block format for [rows][cols] f32. */
PB_API uint32_t pb_quantize_q8_device(const float *x_device, uint32_t rows, uint32_t cols,
                               uint8_t *staging_device, void *stream);
/* RMSNorm (fp32_sse2.rs:1310-1334) of [rows][896] into y; x, w and y 16-byte
 * aligned (PB_CAPACITY otherwise). */
PB_API uint32_t pb_rmsnorm_device(const float *x_device, const float *w_device, uint32_t rows,
                           float *y_device, void *stream);
/* SwiGLU (fp32_sse2.rs:1751-1770) of [rows][4864]. */
PB_API uint32_t pb_swiglu_device(const float *gate_device, const float *up_device, uint32_t rows,
                          float *out_device, void *stream);
/* RoPE on q [rows][896] and k [rows][128] in place at positions[r]
 * (fp32_sse2.rs:1413-1428); v [rows][128]; both written to the KV of slot r. */
PB_API uint32_t pb_rope_kv_device(float *q_device, float *k_device, const float *v_device,
                           const uint32_t *positions_host, uint32_t rows, float *kv_device,
                           uint32_t capacity, uint32_t layer, void *stream);
/* GQA decode attention (fp32_sse2.rs:1430-1672) of q [rows][896] over the KV of
 * slot r at current positions[r]; span (0 = natural) pads the softmax span.
 * capacity and span at most 32768 (the reference's context), capacity a
 * multiple of 4 (PB_CAPACITY otherwise).
 * scores_device (optional) receives [rows][14][span_max] final probabilities. */
PB_API uint32_t pb_attention_device(const float *q_device, const float *kv_device, uint32_t capacity,
                             uint32_t layer, const uint32_t *positions_host, uint32_t rows,
                             uint32_t span, float *out_device, float *scores_device,
                             void *stream);
/* The 8 MiB RoPE table (32768 x 32 x {cos, sin}) the engine uploads; built from
 * glibc powf/cosf/sinf and checked against the reference's SHA-256. */
PB_API uint32_t pb_rope_table(float *table_host);
/* y[i] = the sampler's binary32 exponential of x[i] (bit patterns), the device
 * routine the top-k/top-p weights use: fp32_sse2.rs:378-469 (scalbnf, expf). */
PB_API uint32_t pb_expf_device(const uint32_t *x_device, uint64_t n, uint32_t *y_device, void *stream);

/* --------------------------------------------------- paged serving operators
 * Rotary positions, attention over packed prompts and over a paged cache, and
 * the cache's page operations, for callers that keep their keys and values in
 * pages instead of an engine's slots (no counterpart in the reference, whose
 * rotary table, attention and cache serve one sequence of one model:
 * fp32_sse2.rs:1413-1672, inference.rs:2035-2052).
 *
 * All are asynchronous on `stream`, whose device must be the current one and
 * hold every pointer; none allocates device memory, waits or keeps state (but the
 * count of failures behind pb_attention_status), so they may be captured into a
 * graph and called from any thread.  Arguments that the host can see are checked
 * first: PB_CAPACITY (a size, count or type that is not supported), PB_ALIGNMENT
 * (a pointer or stride), each with its text in pb_last_error_string, and nothing
 * is launched.  What device arrays hold
 * (positions, offsets, page ids, slots, counts) cannot be checked there: values
 * that point outside the buffers described here are ignored as each entry says,
 * never followed.  Operands may not overlap the outputs unless said so. */
enum { PB_TYPE_F32 = 0, PB_TYPE_F16 = 1, PB_TYPE_BF16 = 2 };
/* A position, slot, page id or count of kept nodes that stands for none. */
#define PB_NONE 0xffffffffu
/* Sequences of one attention call. */
#define PB_MAX_SEQS 2048u

/* Rows of heads on the device: element c of head h of row r is data[r *
 * row_stride + h * head_stride + c], strides in elements.  data is 16-byte
 * aligned and both strides are multiples of 16 bytes; those of an output that has
 * several rows or heads are not 0. */
typedef struct pb_rows {
    void *data;
    uint64_t row_stride, head_stride;
} pb_rows;

/* A paged key/value cache on the device: element c of slot s of head h of page p
 * of layer n is k[n * layer_stride + ((p * kv_heads + h) * page_size + s) *
 * head_dim + c], v alike; layer_stride in elements, a multiple of 16 bytes.
 * page_size is 16, 32, 64, 128 or 256; head_dim a multiple of 16 up to 256 (64
 * or 128 for attention); pages * page_size below 2^31. */
typedef struct pb_cache {
    void *k, *v;
    uint64_t layer_stride;
    uint32_t type, layers, pages, page_size, kv_heads, head_dim;
} pb_cache;

/* Rotary positions.  Pair i of the first rotary_dim elements of a head turns by
 * the angle position * f_i, f_i = theta^(-2i / rotary_dim), formed in 64 bits:
 *   a' = m (a cos - b sin), b' = m (b cos + a sin),
 * (a, b) the elements (i, i + rotary_dim / 2) in PB_ROTARY_HALF and (2i, 2i + 1)
 * in PB_ROTARY_INTERLEAVED; the rest of the head stays.  For contexts longer
 * than `original` positions by `factor` (>= 1) the f_i are scaled:
 *   PB_SCALING_LINEAR  f_i / factor;
 *   PB_SCALING_BANDS   with t = original f_i / (2 pi) turns over the original
 *     context: f_i / factor where t <= low, f_i where t >= high, and between
 *     them the mix of both in proportion to t;
 *   PB_SCALING_YARN    the same two ends, mixed in proportion to i between
 *     i0 = floor(d(high)) and i1 = ceil(d(low)), clamped to 0 .. rotary_dim - 1
 *     (i1 = i0 + 0.001 where not above i0), with
 *     d(t) = rotary_dim ln(original / (2 pi t)) / (2 ln theta).
 * m = magnitude; 0 stands for 1, for PB_SCALING_YARN 0.1 ln(factor) + 1.
 * low and high both 0 stand for 1 and 4 (bands) or 1 and 32 (yarn). */
enum { PB_ROTARY_HALF = 0, PB_ROTARY_INTERLEAVED = 1 };
enum { PB_SCALING_NONE = 0, PB_SCALING_LINEAR = 1, PB_SCALING_BANDS = 2, PB_SCALING_YARN = 3 };
typedef struct pb_rotary_config {
    uint32_t head_dim, rotary_dim; /* both multiples of 16, rotary_dim <= head_dim <= 256 */
    uint32_t layout, scaling;
    double theta, factor, original, low, high, magnitude;
} pb_rotary_config;
typedef struct pb_rotary pb_rotary;
/* The frequencies of a configuration, kept on the host: serves any device. */
PB_API uint32_t pb_rotary_create(const pb_rotary_config *config, pb_rotary **out);
PB_API void pb_rotary_destroy(pb_rotary *rotary);
/* q and k [rows] turned by positions_device[row] into q_out and k_out, which may
 * be q and k themselves (the same data and strides).  k_heads 0: no k.  A row
 * whose position is PB_NONE is left out: its outputs stay as they were. */
PB_API uint32_t pb_rotary_device(const pb_rotary *rotary, uint32_t type, uint32_t rows,
                                 const uint32_t *positions_device, uint32_t q_heads,
                                 const pb_rows *q, const pb_rows *q_out, uint32_t k_heads,
                                 const pb_rows *k, const pb_rows *k_out, void *stream);
/* The same, with k turned and v as it is written to `layer` of the cache, whose
 * type, heads and head_dim they have, at slots_device[row] = page * page_size +
 * slot in the page.  A slot outside the cache (PB_NONE) writes no k and v; of
 * rows with the same slot it holds a mix. */
PB_API uint32_t pb_rotary_cache_device(const pb_rotary *rotary, uint32_t rows,
                                       const uint32_t *positions_device, uint32_t q_heads,
                                       const pb_rows *q, const pb_rows *q_out, const pb_rows *k,
                                       const pb_rows *v, const pb_cache *cache, uint32_t layer,
                                       const uint32_t *slots_device, void *stream);

/* Causal attention of packed prompts, out = softmax(scale q k^T) v per head, q
 * head h reading key head h / (q_heads / kv_heads).  Sequence s has the q rows
 * [q_offsets[s], q_offsets[s + 1]) and the key rows [kv_offsets[s], kv_offsets
 * [s + 1]) (kv_offsets NULL: the same), both aligned at their ends: row i of t
 * sees the first n - t + i + 1 of n keys.  A row that sees none, or whose scores
 * are all -inf, is zero; rows behind q_offsets[seqs] stay as they were.  Offsets ascend; they are cut at
 * q_rows and kv_rows.  Keys that a row does not see have no part in it whatever
 * they hold.  head_dim 64 or 128, seqs up to PB_MAX_SEQS, scale positive and scale
 * log2(e) finite. */
PB_API uint32_t pb_prompt_attention_device(uint32_t type, uint32_t head_dim, uint32_t q_heads,
                                           uint32_t kv_heads, uint32_t seqs, uint32_t q_rows,
                                           uint32_t kv_rows, const pb_rows *q, const pb_rows *k,
                                           const pb_rows *v, const pb_rows *out,
                                           const uint32_t *q_offsets_device,
                                           const uint32_t *kv_offsets_device, float scale,
                                           void *stream);

/* Attention of drafted token trees over `layer` of a paged cache.  Sequence s
 * has contexts[s] positions and the rows [offsets[s], offsets[s + 1]) of q, its
 * drafted nodes, whose keys and values stand in the cache behind the context, at
 * position contexts[s] + node.  A node sees the whole context and node j of its
 * sequence where bit j of visible[row] is set (its own bit among them; nodes
 * past 63 are seen by none).  One node with visible 1 is plain decode.  Position
 * p of sequence s is slot p % page_size of page tables[s * table_width + p /
 * page_size]; positions past the table are not seen, a page id outside the cache
 * reads as zeros.  A row that sees nothing is zero; rows behind offsets[seqs]
 * stay as they were.
 * The keys are split over the GPU and joined through `workspace` (16-byte
 * aligned, pb_tree_attention_workspace bytes for the same type, head_dim, heads,
 * seqs and rows); calls that can overlap on the GPU need workspaces of their own. */
PB_API uint64_t pb_tree_attention_workspace(uint32_t type, uint32_t head_dim, uint32_t q_heads,
                                            uint32_t kv_heads, uint32_t seqs, uint32_t rows);
PB_API uint32_t pb_tree_attention_device(const pb_cache *cache, uint32_t layer, uint32_t q_heads,
                                         uint32_t seqs, uint32_t rows, const pb_rows *q,
                                         const pb_rows *out, const uint32_t *tables_device,
                                         uint32_t table_width, const uint32_t *contexts_device,
                                         const uint32_t *offsets_device,
                                         const uint64_t *visible_device, float scale,
                                         void *workspace, uint64_t workspace_bytes, void *stream);

/* Waits for `stream` and reports whether any prompt or tree attention on the current
 * device, on this stream or another, gave up waiting for a copy or a product since the
 * calling host thread last asked, or ever where it has not (PB_DEVICE, once to each
 * thread; the outputs of that attention are not complete).  Not to be called while a graph is captured. */
PB_API uint32_t pb_attention_status(void *stream);

/* Copies page pairs[2 i] to page pairs[2 i + 1] for i < n, keys and values of
 * every layer.  No page may be the target of two pairs or the target of one and
 * the source of another.  Pairs with a page outside the cache are left out. */
PB_API uint32_t pb_cache_copy_pages_device(const pb_cache *cache, uint32_t n,
                                           const uint32_t *pairs_device, void *stream);
/* Keeps the accepted nodes of drafted trees: for every layer, position contexts
 * [s] + nodes[s * nodes_width + i] moves to contexts[s] + i, for i < counts[s]
 * (cut at nodes_width; PB_NONE: none).  nodes ascend within a sequence; an entry below its own
 * index, not above all those before it, or past the table, and a page id outside
 * the cache, is left out.  The pages that are written belong to one sequence each. */
PB_API uint32_t pb_cache_keep_device(const pb_cache *cache, uint32_t seqs,
                                     const uint32_t *tables_device, uint32_t table_width,
                                     const uint32_t *contexts_device,
                                     const uint32_t *counts_device, const uint32_t *nodes_device,
                                     uint32_t nodes_width, void *stream);

/* The host's book of a cache's pages: which pages each sequence holds, counted,
 * so that forked sequences share them.  Host memory only; one thread at a time.
 * A call that fails (PB_CAPACITY: too few free pages or sequences, or an array
 * too short, with the number needed in *needed; PB_STATE: a sequence that is not
 * open) changes nothing. */
typedef struct pb_pool pb_pool;
PB_API uint32_t pb_pool_create(uint32_t pages, uint32_t page_size, uint32_t max_seqs, pb_pool **out);
PB_API void pb_pool_destroy(pb_pool *pool);
/* Opens a sequence without tokens. */
PB_API uint32_t pb_pool_open(pb_pool *pool, uint32_t *seq);
/* Opens a sequence that shares every page of `seq`. */
PB_API uint32_t pb_pool_fork(pb_pool *pool, uint32_t seq, uint32_t *child);
/* Makes room for `tokens` more.  Where the last page is partly filled and
 * shared, the sequence gets a page of its own in its place and pair[0] = the old
 * page, pair[1] = the new one for pb_cache_copy_pages_device, to be run before
 * anything is written; else both are PB_NONE. */
PB_API uint32_t pb_pool_extend(pb_pool *pool, uint32_t seq, uint32_t tokens, uint32_t *pair,
                               uint32_t *needed);
/* Cuts a sequence to `length` tokens and frees the pages behind them. */
PB_API uint32_t pb_pool_truncate(pb_pool *pool, uint32_t seq, uint32_t length);
PB_API uint32_t pb_pool_free(pb_pool *pool, uint32_t seq);
/* Moves the pages in use to the lowest ids: writes n <= capacity pairs (from,
 * to) for pb_cache_copy_pages_device, after which no page past *used is held. */
PB_API uint32_t pb_pool_compact(pb_pool *pool, uint32_t *pairs, uint32_t capacity, uint32_t *n,
                                uint32_t *used, uint32_t *needed);
/* The length of a sequence and its page ids (PB_NONE behind them). */
PB_API uint32_t pb_pool_table(const pb_pool *pool, uint32_t seq, uint32_t *table, uint32_t width,
                              uint32_t *length, uint32_t *needed);
PB_API uint32_t pb_pool_free_pages(const pb_pool *pool);

#ifdef __cplusplus
}
#endif
#endif /* PROMPTBOOT_B200_H */
