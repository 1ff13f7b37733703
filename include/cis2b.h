/* include/cis2b.h -- C ABI of the B200 (sm_100a) CIS-2 deterministic decoder.
 *
 * Drop-in boundary for the reference's model-load / generate / witness
 * surface.  Plain C types only.  Every function returns CIS2B_OK (0) or an
 * error code and never exits the process; the message of the last failure
 * on the calling thread is available from cis2b_last_error().
 *
 * Reference interfaces each entry point replaces (paths inside
 * Aefinity-AI/cis2-lab-archive):
 *   cis2b_load      cis2_model_load()            code/cis2-fp/verify3/model.h:56
 *                   + the load half of main()    code/cis2-fp/gpu/cis2_host.cpp:87-163
 *                                                (config, artifact sha256, table digest,
 *                                                 inv_freq table, bf16 weights)
 *   cis2b_generate  cis2_run_decode()            code/cis2-fp/verify3/model.h:71-76
 *                   + the decode half of main()  code/cis2-fp/gpu/cis2_host.cpp:165-218
 *                   + run_one_prompt (sampled)   code/patches/cis2-fp__cm_e23-pinned-sampling.patch:581-780
 *                   batched over sequences as in code/patches/cis2-fp__cm_gpu3-batched-full.patch:687-763
 *   cis2b_free      cis2_model_free()            code/cis2-fp/verify3/model.h:57
 *   cis2b_info_get  the printed header lines     code/cis2-fp/gpu/cis2_host.cpp:222-227
 *   cis2b_logits    teacher-forced logits        code/cis2-fp/verify3/model.h:138-158
 *                   (cis2_verify_receipt_prefill's all_logits)
 *
 * Threading: a model handle belongs to one device and must not be used by
 * two threads at once (the reference's verify3 state is global and not
 * thread-safe at all, model.c:49).  Different handles are independent.
 */
#ifndef CIS2B_H
#define CIS2B_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CIS2B_OK 0
#define CIS2B_ERR_ARG 1      /* invalid argument or size */
#define CIS2B_ERR_IO 2       /* artifact missing / unreadable / malformed */
#define CIS2B_ERR_CONFIG 3   /* architecture this decoder refuses */
#define CIS2B_ERR_CUDA 4     /* CUDA runtime or kernel failure */
#define CIS2B_ERR_NOMEM 5    /* host or device allocation failed */

#define CIS2B_REDUCTION_SEQUENTIAL 0 /* CIS-2 v0.3b default: strict left-to-right folds */
#define CIS2B_REDUCTION_TREE 1       /* v0.4 candidate: 32-leaf pairwise blocks */

typedef struct cis2b_model cis2b_model;

/* Architecture gate run on config.json before the weights are read.
 * CIS2B_GATE_REFERENCE (0, the default): the Rust reference's gate
 *   (code/cis2-fp/src/main.rs:545-644) key for key and reason for reason:
 *   model_type llama or qwen2, head_dim equal to hidden/heads, ...
 * CIS2B_GATE_QWEN3_PORT (1): the same, but model_type qwen3 is admitted with
 *   its explicit head_dim, as the lab's Qwen3 port of the C++ path decodes it
 *   (labs/w1x-qwen3/scripts/qwen3-port.diff). */
#define CIS2B_GATE_REFERENCE 0
#define CIS2B_GATE_QWEN3_PORT 1

typedef struct {
  int32_t device;        /* CUDA device ordinal */
  int32_t reduction;     /* CIS2B_REDUCTION_* */
  int32_t max_positions; /* prompt + generated positions per sequence; 0 = 4096 */
  int32_t arch_gate;     /* CIS2B_GATE_* */
  int32_t reserved[4];   /* must be zero */
} cis2b_opts;

/* Sampled-mode parameters.  Pass NULL for greedy.
 * scheme CIS2B_SAMPLE_E23 (0): the E23 pinned sampler (SplitMix64 word,
 *   nucleus over the sorted softmax, CDF walk), witness prefix
 *   "CIS2_SAMPLE_V1" before the header; top_k must be 0.
 * scheme CIS2B_SAMPLE_GUMBEL (1): the seeded Gumbel-max clause
 *   "CIS2-SAMPLE-1" (MurmurHash3 noise, top-k then top-p on rank order),
 *   its header absorbed after the prompt ids. */
#define CIS2B_SAMPLE_E23 0
#define CIS2B_SAMPLE_GUMBEL 1
typedef struct {
  uint64_t seed;
  float temperature; /* > 0, finite */
  float top_p;       /* (0, 1]; 1 = disabled */
  uint32_t scheme;   /* CIS2B_SAMPLE_* */
  uint32_t top_k;    /* CIS2B_SAMPLE_GUMBEL only; 0 (or >= vocab) = disabled */
} cis2b_sample;

typedef struct {
  int32_t hidden, intermediate, n_layers, n_heads, n_kv_heads, head_dim, vocab, tied;
  float rms_norm_eps;  /* narrowed once from the f64 config value */
  double rope_theta;
  int32_t reduction;
  int32_t max_positions;
  uint8_t weights_sha256[32];
  uint8_t tokenizer_sha256[32];
  uint8_t config_sha256[32];
  uint8_t table_digest[32];
  uint8_t inv_freq_table_digest[32];
} cis2b_info;

/* Device-side timing of the last cis2b_generate (CUDA events). */
typedef struct {
  double total_ms;    /* first kernel to last witness kernel */
  double prefill_ms;  /* prompt positions through the model */
  double decode_ms;   /* token steps (forward + selection), main stream */
  double witness_tail_ms; /* witness work left after the last decode step */
  int64_t kernel_launches; /* kernels this library launched for the call */
  int64_t h2d_bytes;       /* host -> device bytes copied by the call */
  int64_t d2h_bytes;       /* device -> host bytes copied by the call */
} cis2b_timing;

/* Per-kernel-class CUDA-event timing (for roofline measurement).  Classes: */
#define CIS2B_PROF_LM_HEAD 1u     /* lm_head GEMM (final norm output x vocab) */
#define CIS2B_PROF_LAYER_GEMM 2u  /* q/k/v, o, gate/up and down GEMMs */
#define CIS2B_PROF_ATTENTION 4u   /* scores + softmax + V-mix kernel */
#define CIS2B_PROF_WITNESS 8u     /* witness SHA-256 compression chain */
typedef struct {
  int64_t launches;
  double total_ms;  /* sum of per-launch event durations on the launching stream */
} cis2b_kernel_time;

/* Loads weights_dir/{model.safetensors,config.json,tokenizer.json}: hashes
 * the three artifacts, parses the config (numbers as f64, eps narrowed once),
 * uploads the bf16 weights to the device and builds the pinned inv_freq and
 * RoPE tables there. */
int cis2b_load(const char *weights_dir, const cis2b_opts *opts, cis2b_model **out);

int cis2b_info_get(const cis2b_model *m, cis2b_info *out);

/* Decodes n_seq independent sequences in one batch.
 *   prompt_ids   concatenated prompts (u32 token ids), prompt_lens[n_seq] >= 1
 *   gen_toks     tokens to generate per sequence (>= 0)
 *   sample       NULL = greedy argmax (first maximum wins); else the E23
 *                sampler with position = prompt_len + step
 * Outputs (caller-owned host buffers, any may be NULL except out_witness):
 *   out_tokens        [n_seq][gen_toks]
 *   out_step_digests  [n_seq][gen_toks][32]  witness state finalised after each step
 *   out_witness       [n_seq][32]  final witness digest (CIS2_REF / CIS2_SAMPLE digest)
 *   out_argmax        [n_seq][32]  SHA-256 over prompt ids then generated ids
 * Each sequence's outputs equal its own batch-1 run. */
int cis2b_generate(cis2b_model *m, const uint32_t *prompt_ids, const uint32_t *prompt_lens,
                   uint32_t n_seq, uint32_t gen_toks, const cis2b_sample *sample,
                   uint32_t *out_tokens, uint8_t *out_step_digests, uint8_t *out_witness,
                   uint8_t *out_argmax);

int cis2b_last_timing(const cis2b_model *m, cis2b_timing *out);

/* Times every launch of the classes in `class_mask` (CIS2B_PROF_*) with a
 * CUDA event pair in later cis2b_generate calls; 0 turns it off. */
int cis2b_profile(cis2b_model *m, uint32_t class_mask);
/* Totals of the last cis2b_generate for ONE class bit. */
int cis2b_profile_read(const cis2b_model *m, uint32_t class_bit, cis2b_kernel_time *out);

/* Receipt verification, teacher-forced (replaces cis2_verify_receipt_prefill,
 * code/cis2-fp/verify3/model.h:151-157, and the claim check of
 * verify3/main.c:230-265, batched over sequences).  For each sequence ONE
 * forward pass over prompt + claimed[0 .. gen-2] gives the logits of every
 * claimed step; the token of each step is RECOMPUTED from them (argmax, or
 * the sampler in `sample`) and the witness is rebuilt exactly as
 * cis2b_generate builds it.  An honest claim therefore reproduces the
 * generation's tokens and digests.
 *   claimed           [n_seq][gen]  the receipt's generated ids
 *   out_tokens        [n_seq][gen]  recomputed ids (may be NULL)
 *   out_first_mismatch [n_seq]      first step whose recomputed id differs
 *                                   from the claim, -1 if none (may be NULL)
 *   out_step_digests, out_witness, out_argmax as cis2b_generate. */
int cis2b_verify(cis2b_model *m, const uint32_t *prompt_ids, const uint32_t *prompt_lens, uint32_t n_seq,
                 const uint32_t *claimed, uint32_t gen_toks, const cis2b_sample *sample, uint32_t *out_tokens,
                 int32_t *out_first_mismatch, uint8_t *out_step_digests, uint8_t *out_witness,
                 uint8_t *out_argmax);

/* Teacher-forced logits of ONE sequence: runs ids[0 .. n_prompt+n_rows-2]
 * and writes the fp32 logits after positions n_prompt-1 .. n_prompt+n_rows-2
 * into out_logits[n_rows][vocab]. */
int cis2b_logits(cis2b_model *m, const uint32_t *ids, uint32_t n_prompt, uint32_t n_rows,
                 float *out_logits);

/* Per-op trace, for localising a parity failure (debug only; the
 * reference CLI's --trace F, code/cis2-fp/gpu/cis2_host.cpp:76, 173-193, and
 * its emit points, gpu/cis2_model.h:482-496, 685-760).  Runs ids[0 .. n_ids)
 * as ONE sequence, position by position, and writes one line per op output
 *   pos=P layer=L op=NAME sha256=HEX
 * (SHA-256 over the output's fp32 bits, u32 LE) in the reference's op order:
 * embedding; per layer norm1 q k v [q_norm k_norm] rope_q rope_k scores
 * softmax attn_out o_proj resid1 norm2 gate up silu_mul down resid2; then
 * final_norm and logits.  To trace a generation of G tokens as the
 * reference does, pass the prompt followed by the G generated ids. */
int cis2b_trace(cis2b_model *m, const uint32_t *ids, uint32_t n_ids, const char *trace_path);

void cis2b_free(cis2b_model *m);

/* Message of the last failed call on this thread ("" if none). */
const char *cis2b_last_error(void);

/* ---- kernel-level entry points (host buffers in and out) ---------------
 * Used by the parity tests to check single kernels against the CPU oracle. */

/* y[i] = f(x[i]); f: 0 exp, 1 sin, 2 cos, 3 ln, 4 silu, 5 rsqrt (spec §6). */
int cis2b_op_pinned_map(int32_t device, int32_t fn, const float *x, float *y, size_t n);
/* Y[r][o] = dot(W[o,:], X[r,:]) in the pinned order; W bf16 [n_out][k], k % 8 == 0.
 * reduction: CIS2B_REDUCTION_SEQUENTIAL or _TREE through the panel kernel the
 * prompt pass uses, or CIS2B_OP_MATMUL_DECODE / _DECODE_TREE: sequential or
 * tree order through the few-row kernel decode steps use (rows <= 1024; tree
 * order: k % 32 == 0). */
#define CIS2B_OP_MATMUL_DECODE 2
#define CIS2B_OP_MATMUL_DECODE_TREE 3
int cis2b_op_matmul(int32_t device, const uint16_t *W, const float *X, int32_t rows, int32_t n_out,
                    int32_t k, int32_t reduction, float *Y);
/* Index (0-based) of the register tile the many-row product picks for
 * rows x n_out (sequential order, rows >= 64), or -1; lets the parity tests
 * confirm that their shapes reach every tile of that kernel. */
int cis2b_op_gemm_tile(int32_t rows, int32_t n_out);
/* Witness stream check: absorbs `prefix` (byte path), then n_chunks chunks of
 * chunk_words u32 words through the device step path (last word of each
 * chunk plays the token id); writes the digest after each chunk. */
int cis2b_op_sha256_stream(int32_t device, const uint8_t *prefix, size_t prefix_len,
                           const uint32_t *words, uint32_t chunk_words, uint32_t n_chunks,
                           uint8_t *out_digests);
/* Greedy token selection on `rows` logits rows of n values each, through
 * the kernel the decode steps use: the first index of the strict maximum
 * (code/cis2-fp/src/main.rs:1161-1169; gpu/cis2_model.h:764-774), so an
 * exact tie -- +0 against -0 included -- keeps the lower index, a NaN at
 * index 0 selects 0 and a NaN elsewhere is never selected. */
int cis2b_op_argmax(int32_t device, const float *logits, int32_t rows, int32_t n, uint32_t *out_index);
/* E23 sampler on one logits row; position < 2^31. */
int cis2b_op_sample(int32_t device, const float *logits, int32_t n, float temperature, float top_p,
                    uint64_t seed, uint64_t position, uint32_t *out_index);
/* Seeded Gumbel-max ("CIS2-SAMPLE-1") draw on one logits row; step is the
 * 0-based generation step. */
int cis2b_op_sample_gumbel(int32_t device, const float *logits, int32_t n, float temperature, uint32_t top_k,
                           float top_p, uint64_t seed, uint32_t step, uint32_t *out_index);

/* No counterpart in the reference.  The E23 sampler on one logits row that
 * ALLOCATES NOTHING: for callers that cannot call cudaMalloc -- code whose
 * device memory is owned by its own allocator (a framework's caching pool,
 * a pre-reserved arena) that must not be bypassed, or code on a
 * latency-critical path where cudaMalloc/cudaFree would synchronise the
 * device.  The caller passes device pointers for the input row and the
 * output index; the sampler's working memory is a fixed array inside the
 * library (5 floats per logit for CIS2B_STATIC_SAMPLE_MAX logits, about
 * 5 MiB) that every GPU which loads the library keeps until the process
 * exits.
 *   d_logits     device pointer to n fp32 logits, 1 <= n <= CIS2B_STATIC_SAMPLE_MAX
 *   d_out_index  device pointer to one uint32, written with the drawn index
 *   stream       cudaStream_t to run on (NULL: the legacy default stream)
 *   position     < 2^31
 * Makes `device` current on the calling thread.  The first call on a device
 * looks up the array's device address and keeps it; make that first call
 * before any stream capture.  A device reset that destroys the primary
 * context (cudaDeviceReset) makes the kept address stale: do not call this
 * entry point again in that process afterwards.  The call is asynchronous:
 * the index is valid once `stream` has reached it.  All calls on one device
 * in one process share the one array, whichever model handle or thread
 * makes them, and it keeps the last call's contents (every element the
 * sampler reads it writes first), so calls whose work overlaps on the GPU --
 * two streams, or two threads -- race and must be ordered by the caller.
 * Only this entry point uses the array: it never races with cis2b_generate,
 * cis2b_verify or the other entry points, and separate processes each have
 * their own copy.  Sizes above the maximum are rejected with CIS2B_ERR_ARG.
 * Same result as cis2b_op_sample. */
#define CIS2B_STATIC_SAMPLE_MAX 262144
int cis2b_op_sample_static(int32_t device, const float *d_logits, int32_t n, float temperature, float top_p,
                           uint64_t seed, uint64_t position, uint32_t *d_out_index, void *stream);

/* ---- 4-bit key/value cache ----------------------------------------------
 * No counterpart in the reference.  A paged cache that holds keys and values
 * in 4 bits, for callers that run their own layers: the step's block tables
 * and slot maps built on the GPU, rows quantised into the cache and read
 * back, and causal attention over it with an optional sliding window and
 * sinks.  Results are approximate (4 bits) and outside the witness; every
 * call is deterministic: the same inputs give the same bits.
 *
 * These entry points take DEVICE pointers, run asynchronously on `stream`
 * (NULL: the legacy default stream), allocate nothing and can be captured in
 * a CUDA graph.  They make the cache's device current on the calling thread.
 *
 * Format.  A group is one token's head_dim elements of one KV head:
 *   base = min(x) rounded down to bfloat16
 *   step = (max(x) - base) / 15 rounded up to bfloat16, 0 if below 2^-100
 *   code = rint((x - base) * (1 / step)) clamped to 0..15, 0 if step is 0
 * each operation rounded to fp32; a code stands for base + step * code.  A
 * group with a NaN or an infinity, or whose range passes fp32's, reads back
 * as NaN.  Per page and KV head the pool holds page_size / 16 records of 16
 * tokens: 16 x head_dim/2 bytes of key codes (byte b: element 2b in the low
 * four bits, 2b + 1 in the high), the same of value codes, then 16 x {key
 * step, key base, value step, value base} as bfloat16. */
#define CIS2B_F32 0
#define CIS2B_F16 1
#define CIS2B_BF16 2

typedef struct {
  int32_t device;
  int32_t pages;     /* >= 1; pages * page_size < 2^31 */
  int32_t page_size; /* tokens: 16, 32, 64, 128 or 256 */
  int32_t kv_heads;  /* >= 1 */
  int32_t head_dim;  /* 64 or 128 */
  int32_t reserved;  /* must be zero */
  void *pool;        /* cis2b_kv4_bytes() bytes, 16-byte aligned */
  int32_t *status;   /* one word or NULL: bits OR-ed in by the kernels, below */
} cis2b_kv4_cache;

#define CIS2B_KV4_BAD_SLOT 1 /* a slot >= pages * page_size; the row was skipped */
#define CIS2B_KV4_STUCK 4    /* a wait inside a kernel ran out; the call's results are not valid */
#define CIS2B_KV4_BAD_PAGE 2 /* a visible key on a page that is not in the pool; it was not seen */

/* Bytes of the pool: pages * kv_heads * page_size * (head_dim + 8). */
int cis2b_kv4_bytes(const cis2b_kv4_cache *c, uint64_t *out_bytes);

/* Plans one step of a batch: request r holds cached[r] tokens and adds
 * new_tokens[r] (0 or more).  Its rows are row_start[r] .. row_start[r+1]-1
 * of the step's tensors, in request order.  Pages that it needs beyond
 * ceil(cached / page_size) are taken from free_pages in request order and
 * entered in its row of `table`; other entries are left as they are.
 *   length     [requests]      cached + new_tokens
 *   row_start  [requests + 1]  prefix sums of new_tokens
 *   slot, position, request [rows]  of each row: page * page_size + offset in
 *              the cache, position in the request, request; -1 in the rows
 *              past row_start[requests]
 *   counts     [4]  rows in use, pages needed, CIS2B_KV4_PLAN_* bits, 0
 * A row whose page is missing (bits FREE, WIDTH) has slot -1.  At most 16384
 * requests.  Work that a later call must see goes on the same stream. */
#define CIS2B_KV4_PLAN_FREE 1     /* more pages needed than free_count */
#define CIS2B_KV4_PLAN_WIDTH 2    /* a request longer than width * page_size */
#define CIS2B_KV4_PLAN_ROWS 4     /* more new tokens than `rows` */
#define CIS2B_KV4_PLAN_NEGATIVE 8 /* a negative cached or new_tokens; taken as 0 */
typedef struct {
  int32_t device;
  int32_t requests;   /* 1 .. 16384 */
  int32_t rows;       /* capacity of slot, position and request; >= 0 */
  int32_t width;      /* entries per row of table */
  int32_t page_size;  /* 16, 32, 64, 128 or 256 */
  int32_t free_count; /* entries of free_pages */
  const int32_t *cached, *new_tokens; /* [requests] */
  const int32_t *free_pages;          /* [free_count]; may be NULL if 0 */
  int32_t *table;                     /* [requests][width] */
  int32_t *length, *row_start;
  int32_t *slot, *position, *request; /* may be NULL if rows is 0 */
  int32_t *counts;
} cis2b_kv4_step;
int cis2b_kv4_plan(const cis2b_kv4_step *s, void *stream);

/* Quantises rows k, v [rows][kv_heads][head_dim] (elements of a head
 * contiguous; row and head strides in elements) into their slots.  A
 * negative slot skips its row.  Slots in one call must differ. */
int cis2b_kv4_append(const cis2b_kv4_cache *c, int32_t dtype, const void *k, const void *v,
                     int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                     const int32_t *slot, int32_t rows, void *stream);
/* Reads the rows of `slot` back as the values that their codes stand for,
 * into contiguous k, v [rows][kv_heads][head_dim]; zeros for negative slots
 * and slots out of range. */
int cis2b_kv4_gather(const cis2b_kv4_cache *c, int32_t dtype, void *k, void *v, const int32_t *slot, int32_t rows,
                     void *stream);

/* Causal attention of the step's rows over the cache (their own keys and
 * values appended before).  Row i of request r stands at position
 * p = length[r] - (row_start[r+1] - row_start[r]) + i - row_start[r] and sees
 * keys j <= p with, if window > 0, j > p - window or j < sinks.  Query head h
 * reads KV head h / (heads / kv_heads).  Rows that see nothing, and rows past
 * row_start[requests], are zero.
 *   max_new    the most rows of any one request, or a bound (chooses the
 *              kernel; a request with more is still computed)
 *   scale      factor of the scores (1 / sqrt(head_dim) in most models)
 *   flags      0: the keys of all requests are shared out evenly over the
 *              GPU, so the grouping of a row's sums goes by the whole batch;
 *              CIS2B_KV4_WHOLE: a row's sums are grouped by its own request
 *              alone, and a request's result does not depend on the others
 *              (given the same max_new), at the cost of parallelism over long
 *              requests
 *   work       cis2b_kv4_workspace() bytes or more, of which the first
 *              CIS2B_KV4_WORK_ZERO are zeroed once before the first call;
 *              then left alone: calls of other sizes may use
 *              it too, but calls that may overlap on the GPU (replays of
 *              captured ones among them) need one each.
 *              Zero it again after CIS2B_KV4_STUCK
 * Softmax statistics and sums are held in fp32 (of bf16 rows in the kernel for
 * one or few tokens, the tensor cores' sums keep about 15 bits).  The tensor cores
 * cut off what falls below a sum's last bit, which adds up where values have one
 * sign: fp32 rows over 32,768 (131,072) such keys are off by 2e-5 (1e-4) up to 32
 * query columns and 2e-4 (9e-4) from there on with CIS2B_KV4_WHOLE, by 5e-7 and
 * 6e-6 in parts.  Codes are
 * exact; a row's query elements and its weights are rounded to 22 bits (fp32
 * rows) or 11 (16-bit rows), those below 2^-10 (22 bits) or 2^-21 (11 bits) of
 * the row's largest to 2^-32 of it.  What a row does not see, whatever finite
 * or other number stands there, changes no bit of its result; a query row with
 * an infinity or a NaN is NaN where it sees anything.  Queries of 2^120 and keys
 * of 2^118 and more may make a NaN: sums on the way to their scores may pass
 * fp32's range. */
#define CIS2B_KV4_WHOLE 1
#define CIS2B_KV4_WORK_ZERO 266240
typedef struct {
  int32_t dtype;    /* CIS2B_F32, _F16 or _BF16: q and out */
  int32_t heads;    /* a multiple of kv_heads, at most 32 times as many */
  int32_t requests; /* >= 1; (requests + rows) * kv_heads <= 2^30 */
  int32_t rows;     /* rows of q and out */
  int32_t width;    /* entries per row of table */
  int32_t max_new;  /* >= 1 */
  int32_t window;   /* 0: none */
  int32_t sinks;    /* >= 0 */
  float scale;
  int32_t flags;    /* CIS2B_KV4_WHOLE or 0 */
  const void *q;
  void *out;        /* [rows][heads][head_dim]; strides in elements, heads' elements contiguous */
  int64_t q_row_stride, q_head_stride, out_row_stride, out_head_stride;
  const int32_t *table, *length, *row_start;
  void *work;       /* 16-byte aligned */
  uint64_t work_bytes;
} cis2b_kv4_attn;
int cis2b_kv4_workspace(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, uint64_t *out_bytes);
int cis2b_kv4_attention(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, void *stream);

/* ---- drafted trees and encoders over the 4-bit cache ---------------------
 * Rows that do not see by their place alone: the tokens of a tree that a
 * smaller model has drafted, and rows that attend to an encoder's states.
 *
 * A step of drafted tokens.  cis2b_kv4_plan gives request r's n = row_start[r+1]
 * - row_start[r] new tokens the places that follow its cached = length[r] - n
 * tokens, in row order.  Row 0 of a request is the token that the model has
 * settled on last; parent[row] is the number, within the request, of the row
 * that a row continues, or -1 for one that continues the cached tokens.  A
 * parent stands before its children.  Then: cis2b_kv4_plan_tree (of layers with a
 * window cis2b_kv4_plan_tree_window) for masks and positions; per layer cis2b_kv4_append and cis2b_kv4_tree_attention; when the
 * model's own next token after every row is known, cis2b_kv4_accept, and
 * cis2b_kv4_keep on the caches of all layers.  Next step's `cached` is kept[].
 * All entry points follow the rules above: device pointers, asynchronous,
 * nothing allocated, capturable, deterministic. */
#define CIS2B_KV4_TREE_MOST 1024 /* rows of one request's tree; those past it are no part of it */
#define CIS2B_KV4_TREE_PARENT 1  /* a parent < -1 or not before its child; taken as -1 */
#define CIS2B_KV4_TREE_ROWS 2    /* a request with more rows than the masks (or CIS2B_KV4_TREE_MOST) hold */

/* Masks and positions of drafted tokens.  Bit b % 32 of mask[row][b / 32] is
 * set for row b of the request being the row itself or one of its ancestors;
 * position[row] = cached + number of its ancestors.  Rows past 32 * words of
 * their request, and rows past row_start[requests], get an empty mask and
 * position -1. */
typedef struct {
  int32_t device;
  int32_t requests; /* >= 1 */
  int32_t rows;     /* of parent, mask and position */
  int32_t words;    /* of a row of mask: 1 .. 32 */
  const int32_t *length, *row_start, *parent;
  int32_t *mask;     /* [rows][words] */
  int32_t *position; /* [rows] */
  int32_t *status;   /* one word or NULL: CIS2B_KV4_TREE_* bits OR-ed in */
} cis2b_kv4_tree;
int cis2b_kv4_plan_tree(const cis2b_kv4_tree *t, void *stream);
/* The same for layers with a sliding window: a row's mask leaves out the
 * ancestors that stand `window` or more positions before it and are not among
 * the first `sinks` positions, as causal attention of the text along the path
 * would.  window 0: none.  Positions are the same.  Where no path is longer than
 * the window the masks are cis2b_kv4_plan_tree's; where one is, layers with
 * different windows need masks of their own. */
int cis2b_kv4_plan_tree_window(const cis2b_kv4_tree *t, int32_t window, int32_t sinks, void *stream);

/* The longest path of drafted tokens that the model agrees with.  target[row]
 * is the model's next token after that row (greedy, or drawn by a sampler
 * whose randomness goes by seed and position).  The path begins at row 0 and
 * goes on, from row i, to the lowest row whose parent is i and whose token is
 * target[i], as long as there is one.
 *   accepted   [requests]  rows of the path: >= 1, or 0 for a request without rows
 *   path       [rows]      path[row_start + k] is its k-th row within the
 *              request; -1 from accepted on, and past row_start[requests]
 *   next_token [requests]  target of its last row; -1 for a request without rows
 *   kept       [requests]  cached + accepted */
typedef struct {
  int32_t device;
  int32_t requests; /* >= 1 */
  int32_t rows;
  int32_t reserved; /* must be zero */
  const int32_t *length, *row_start, *token, *parent, *target;
  int32_t *accepted, *path, *next_token, *kept;
  int32_t *status; /* as above */
} cis2b_kv4_draft;
int cis2b_kv4_accept(const cis2b_kv4_draft *d, void *stream);

/* Moves, in each of n caches (of one device, page_size, kv_heads and
 * head_dim), what slot[row_start + path[k]] holds to slot[row_start + k], for
 * every request and k < accepted: bit for bit, all moves at once.  path[k] >=
 * k; the slots of one call differ.  Entries with a slot < 0 are skipped, as
 * are, with CIS2B_KV4_BAD_SLOT or CIS2B_KV4_BAD_PATH in the caches' status,
 * those out of range. */
#define CIS2B_KV4_BAD_PATH 8 /* path[k] < k, or not a row of the request */
typedef struct {
  int32_t device;
  int32_t requests; /* >= 1 */
  int32_t rows;
  int32_t reserved; /* must be zero */
  const int32_t *row_start, *accepted, *path, *slot;
} cis2b_kv4_kept;
int cis2b_kv4_keep(const cis2b_kv4_cache *caches, int32_t n, const cis2b_kv4_kept *k, void *stream);

/* Attention of drafted tokens.  Row i of request r sees of its cached tokens
 * (j < cached) all, or with window > 0 those with j > position[i] - window or
 * j < sinks, and of its new ones those whose bit is set in mask[i] (no more
 * than 32 * words, none at or past length[r]), whatever the window: which of its
 * ancestors a window hides is in the mask (cis2b_kv4_plan_tree_window).  position
 * is read with window > 0 only; one outside cached .. cached + n - 1 counts as
 * the nearest inside.  Any bits may be set: a tree's, or another order of the
 * new tokens among themselves.  Everything else as cis2b_kv4_attention, but for
 * the precision of two kinds of rows.  bfloat16 rows, where a request has 17 query
 * columns (rows x heads / kv_heads) or more: every key and value is taken times a
 * power of two of its own and rounded to 11 bits, no token's size mattering to
 * another's; weights below 2^-18 of the row's largest are rounded to 2^-28 of it.
 * (Without CIS2B_KV4_WHOLE rows of 65 to 128 columns are such rows or not by the
 * number of requests and the tables' width, too.)
 * fp32 rows: the products of 16 keys are summed as the tensor cores do, which cut
 * off what falls below fp32's last bit; the sums over those are rounded to fp32. */
int cis2b_kv4_tree_attention(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, const int32_t *mask, int32_t words,
                             const int32_t *position, void *stream);
/* Attention to an encoder's states: every row of request r sees the first
 * length[r] tokens of its table, 0 or more, however many rows it has; nothing
 * is causal.  window and sinks must be 0.  Requests may share pages.  Everything
 * else as cis2b_kv4_tree_attention. */
int cis2b_kv4_cross_attention(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, void *stream);
/* Bytes of `work` for either of the two. */
int cis2b_kv4_tree_workspace(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, uint64_t *out_bytes);

#ifdef __cplusplus
}
#endif
#endif /* CIS2B_H */
