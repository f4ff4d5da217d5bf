/*
 * jv.h — C ABI of the B200 Jevstral forward pass.
 *
 * The .NET host keeps its public API (JevstralDecider, VerdictScorer, SystemPromptCache,
 * the `jev` CLI) and replaces the body of MinistralModel and KvCache with P/Invoke calls
 * into this library. Every entry point below names the reference member it replaces
 * (paths inside theolivenbaum/llm-shield). Signatures hold plain pointers and sizes only.
 *
 * Threading: a jv_model (weights on one GPU) may be shared by several jv_ctx; a jv_ctx
 * (one KV cache, one CUDA stream, activation buffers) is single-threaded, like a
 * MinistralModel instance (src/Jevstral/Model/MinistralModel.cs:21-22).
 *
 * Errors: every int-returning call returns a JV_* status. jv_last_error() gives the
 * calling thread's last message. The C# binding maps codes back to the exception types
 * the reference throws (src/Jevstral/Model/MinistralModel.cs:202,207,306;
 * src/Jevstral/Numerics/QuantMatMul.cs:300-302; src/Jevstral/Model/KvCache.cs:96-97,118-120;
 * src/Jevstral/Gguf/GgufFile.cs:156-172).
 */
#ifndef JV_H
#define JV_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum jv_status {
    JV_OK = 0,
    JV_ERR_ARG = 1,            /* ArgumentException / ArgumentNullException          */
    JV_ERR_RANGE = 2,          /* ArgumentOutOfRangeException                        */
    JV_ERR_FORMAT = 3,         /* InvalidDataException / KeyNotFoundException         */
    JV_ERR_IO = 4,             /* IOException / FileNotFoundException                 */
    JV_ERR_UNSUPPORTED = 5,    /* NotSupportedException                              */
    JV_ERR_CANCELLED = 6,      /* OperationCanceledException                         */
    JV_ERR_DEVICE = 7,         /* a CUDA call failed                                 */
    JV_ERR_DEVICE_TIMEOUT = 8, /* a bounded device-side wait gave up                 */
    JV_ERR_OOM = 9,            /* device memory exhausted                            */
    JV_ERR_NUMERIC = 10        /* an activation left the fp16 range of the device path
                                  (|x| >= 65520 or not a number): ArithmeticException.
                                  The reference's fp32 path has no such limit.        */
};

typedef struct jv_model jv_model;       /* weights resident on one device            */
typedef struct jv_ctx jv_ctx;           /* MinistralModel instance: KV cache + stream */
typedef struct jv_snapshot jv_snapshot; /* refcounted KV pages of a prefix            */
typedef struct jv_server jv_server;     /* many requests over one 8-bit KV cache      */

/* ModelConfig (src/Jevstral/Model/ModelConfig.cs:11-56), plus the resolved RoPE magnitude
 * scale (Rope.MagnitudeScale, src/Jevstral/Model/Rope.cs:28) and the weight type. */
typedef struct jv_config {
    int32_t layers, hidden, heads, kv_heads, head_dim, ff, vocab, rope_dim;
    int32_t context_length, rope_orig_ctx, yarn_active, weight_type;
    float eps, rope_base, rope_scale, rope_mscale, temperature_scale;
} jv_config;

/* TokenLayout (src/Jevstral/Model/MinistralModel.cs:703-718): token t is written to KV slot
 * slot[t], rotated as position[t], and sees slots [0, shared[t]) and [segment[t], slot[t]].
 * outputs[] are the token indices whose logits are returned; end is one past the highest
 * slot written; sparse is carried for fidelity (it only picks a CPU loop in the reference). */
typedef struct jv_layout {
    const int32_t* slot;
    const int32_t* position;
    const int32_t* shared;
    const int32_t* segment;
    const int32_t* outputs;
    int32_t n_outputs;
    int32_t end;
    int32_t sparse;
} jv_layout;

/* IActivationSink.Observe (src/Jevstral/Model/MinistralModel.cs:787-790). Called
 * synchronously with host fp32 data named as the reference names them: "embeddings",
 * "blk.{l}.attn_norm|q_rope|k_rope|v|attn_weighted|attn_out|post_attn|ffn_norm|ffn_out|output",
 * "final_norm", "logits". */
typedef void (*jv_activation_sink)(void* user, const char* name, const float* values, int32_t rows,
                                   int32_t cols);

/* ---- library / device -------------------------------------------------------------- */

const char* jv_last_error(void);
int jv_device_count(int32_t* count);
/* Counts this library's kernel launches on the calling process (all contexts). */
int64_t jv_kernel_launches(void);
/* How this copy of the library was built (no counterpart in the reference): bit 0 set in the
 * bounds-checked build (libjv_checked.so), whose kernels test every KV page-table lookup and
 * GEMM work unit and fail the call with JV_ERR_RANGE, naming the site, instead of touching
 * memory out of range. The check stands in for a memory checker; it is slower and not for
 * serving. */
#define JV_FEATURE_BOUNDS_CHECK 1
int32_t jv_build_features(void);

/* ---- model (weights) ----------------------------------------------------------------- */

/* new MinistralModel(ggufPath) weight binding (MinistralModel.cs:56-123), GgufFile parsing
 * (src/Jevstral/Gguf/GgufFile.cs:76-172) and ModelConfig.FromGguf (ModelConfig.cs:62-112).
 * Copies the quantized blocks of every matrix to `device` once, re-tiled but bit-identical.
 * kv_pool_mb sizes the device KV page pool (0 = default). */
int jv_model_open(const char* gguf_path, int32_t device, int32_t kv_pool_mb, jv_model** out);
void jv_model_close(jv_model* model);
/* MinistralModel.Config (MinistralModel.cs:48). */
int jv_model_config(const jv_model* model, jv_config* out);

/* ---- context (MinistralModel instance state) ---------------------------------------- */

/* The KvCache + logits buffer a MinistralModel owns (MinistralModel.cs:100-101). */
int jv_ctx_create(jv_model* model, int32_t initial_capacity, jv_ctx** out);
void jv_ctx_destroy(jv_ctx* ctx);
/* Activation capture (the IActivationSink argument of ForwardAsync, MinistralModel.cs:155). */
int jv_ctx_set_sink(jv_ctx* ctx, jv_activation_sink sink, void* user);
/* ParallelOptions.CancellationToken: when *flag becomes non-zero the forward stops between
 * layers and returns JV_ERR_CANCELLED (KernelTests.cs:206-218). NULL clears it. */
int jv_ctx_set_cancel(jv_ctx* ctx, const volatile int32_t* flag);
/* The cudaStream_t every kernel of this context runs on (for event timing). */
void* jv_ctx_stream(jv_ctx* ctx);

/* Per-kernel-class timing with CUDA events on the context's stream (no counterpart in the
 * reference, which times with a Stopwatch around whole calls, src/Jevstral.Cli/Benchmark.cs:549-623).
 * While enabled every launch of the class is bracketed by events; totals accumulate until
 * reset. kind: 0 tensor-core GEMM, 1 GEMV, 2 attention, 3 everything else. flops/bytes are
 * the algorithmic work of the timed launches. */
enum jv_profile_kind { JV_PROF_GEMM = 0, JV_PROF_GEMV = 1, JV_PROF_ATTENTION = 2, JV_PROF_OTHER = 3 };
int jv_ctx_profile(jv_ctx* ctx, int32_t enable);
int jv_ctx_profile_read(jv_ctx* ctx, int32_t kind, double* total_ms, int64_t* launches, double* flops, double* bytes);
int jv_ctx_profile_reset(jv_ctx* ctx);

/* Check of the device-timeout path (no counterpart in the reference, which has no device
 * waits): runs one kernel whose bounded wait nothing completes. The wait gives up after
 * bound_cycles SM clock cycles (0 < bound_cycles <= 4e9; the tensor-core kernels use 4e9,
 * about 2 s), and the call returns JV_ERR_DEVICE_TIMEOUT with the wait named in
 * jv_last_error(). The context stays usable: its error word is cleared and later calls run
 * normally. Nothing faults or hangs. */
int jv_ctx_check_wait_timeout(jv_ctx* ctx, int64_t bound_cycles);

/* ---- forward passes ------------------------------------------------------------------- */

/* MinistralModel.ForwardAsync(tokens, options) (MinistralModel.cs:139) — appends tokens and
 * writes the full-vocabulary logits of the last position to logits[vocab]. With logits ==
 * NULL this is PrefillAsync (MinistralModel.cs:148): KV only, no LM head. */
int jv_forward(jv_ctx* ctx, const int32_t* tokens, int32_t n, float* logits);

/* MinistralModel.ForwardSelectedAsync (MinistralModel.cs:165-172): appends tokens; out[n_rows]
 * = logits of vocab rows `rows` at the last position. */
int jv_forward_selected(jv_ctx* ctx, const int32_t* tokens, int32_t n, const int32_t* rows,
                        int32_t n_rows, float* out);

/* MinistralModel.ForwardTreeAsync (MinistralModel.cs:198-219); ForwardBranchesAsync
 * (MinistralModel.cs:187) when n_trunk == 0. branch_tokens holds the branches back to back
 * (branch_lengths[b] tokens each). out[n_branches][n_rows] = logits of `rows` at each
 * branch's last token. The branch tokens stay in the KV cache, as in the reference. */
int jv_forward_tree(jv_ctx* ctx, const int32_t* trunk, int32_t n_trunk, const int32_t* branch_tokens,
                    const int32_t* branch_lengths, int32_t n_branches, const int32_t* rows,
                    int32_t n_rows, float* out);

/* Many independent ForwardTreeAsync decisions in one pass: the batch entry of the data-parallel
 * path (no single reference member; each decision is what MinistralModel.cs:198-219 computes
 * for its trunk and branches on an empty cache). Decision d has trunk_lengths[d] trunk tokens
 * and branch_counts[d] branches; `tokens` holds each decision's trunk and then its branches,
 * decision after decision, and branch_lengths every branch in that order. A decision sees only
 * its own tokens (not the cache's contents, not the other decisions). out[sum of branch_counts]
 * [n_rows] = logits of `rows` at each branch's last token, in branch order; each row is
 * bit-identical to that decision run alone by jv_forward_tree on an empty cache. The cache is
 * left as it was (its length is restored after the pass). */
int jv_decide_batch(jv_ctx* ctx, int32_t n_decisions, const int32_t* tokens, const int32_t* trunk_lengths,
                    const int32_t* branch_counts, const int32_t* branch_lengths, const int32_t* rows,
                    int32_t n_rows, float* out);

/* The private ForwardAsync(tokens, capture, options, computeLogits, layout, selectedRows,
 * selectedOut) every public overload funnels into (MinistralModel.cs:301-435).
 * layout == NULL means a causal append at the cache end. With rows != NULL, out receives
 * [n_outputs][n_rows] selected logits; with rows == NULL and full_vocab != 0, out receives
 * [n_outputs][vocab] (ForwardTreeLogitsAsync / ForwardRowsAsync, MinistralModel.cs:227-294);
 * with compute_logits != 0, logits receives the last position's full vocabulary. */
int jv_forward_layout(jv_ctx* ctx, const int32_t* tokens, int32_t n, const jv_layout* layout,
                      const int32_t* rows, int32_t n_rows, int32_t full_vocab, float* out,
                      int32_t compute_logits, float* logits);

/* The benchmark's decode loop (src/Jevstral.Cli/Benchmark.cs:411-422): `steps` single-token
 * forwards with the full LM head, each feeding back the argmax
 * (Kernels.ArgMax, src/Jevstral/Numerics/Kernels.cs:146) of the previous one, starting from
 * first_token. Writes the chosen tokens to out_tokens[steps]. */
int jv_decode_greedy(jv_ctx* ctx, int32_t first_token, int32_t steps, int32_t* out_tokens);

/* ---- QuantMatMul on device buffers (src/Jevstral/Numerics/QuantMatMul.cs) -------------
 * A quantized matrix lives on the device in this library's re-tiled layout (the GGUF blocks
 * of 128 rows x 64 columns gathered into one contiguous chunk; bits unchanged). All pointers
 * below are device pointers; stream is a cudaStream_t (NULL = the legacy default stream).
 * type is the GGML type id: 8 Q8_0, 7 Q5_1, 2 Q4_0. rows % 128 == 0, cols % 64 == 0. */

/* Bytes of the re-tiled layout (WeightMatrix, src/Jevstral/Numerics/WeightMatrix.cs:16-66). */
int64_t jv_qweight_bytes(int32_t type, int32_t rows, int32_t cols);
/* Re-tile `rows` GGUF rows (GgmlTypeInfo.RowBytes(type, cols) bytes each, back to back) into
 * `tiled` (jv_qweight_bytes bytes). */
int jv_qweight_pack(int32_t type, const void* gguf_rows, int32_t rows, int32_t cols, void* tiled, void* stream);
/* QuantMatMul.ForwardAsync for one token (QuantMatMul.cs:127-129 -> RunRowsFloat :140-176):
 * y[rows] = W x[cols] with W decoded to fp32 exactly as Dequantizer does and fp32 FMA. Uses a
 * split-K partial buffer that it allocates on the device on first use (and keeps). */
int jv_qmatvec(int32_t type, const void* tiled, int32_t rows, int32_t cols, const float* x, float* y, void* stream);
/* jv_qmatvec without any device allocation. No counterpart in the reference: it is for
 * callers that must not allocate device memory on the call path (a host that has planned
 * all of HBM up front, or one running under a memory cap owned by another component). The
 * split-K partials live in a fixed 1 MiB device array (JV_QMATVEC_SCRATCH_FLOATS_MAX = 262144
 * floats) built into the library; a call needs splits x rows floats (splits as jv_qmatvec
 * picks them) and fails with JV_ERR_RANGE above that. All calls on a device share the array:
 * nothing in it has to start at zero, but calls that overlap in time on one device race, so
 * serialize them. The first call on each device does a one-time set-up (a symbol-address
 * lookup with that device current); make it before any stream capture begins. */
#define JV_QMATVEC_SCRATCH_FLOATS_MAX 262144
int jv_qmatvec_noalloc(int32_t type, const void* tiled, int32_t rows, int32_t cols, const float* x, float* y,
                       void* stream);

/* ---- paged batches: many requests in one 8-bit KV cache, on device buffers -------------
 * The operators a server runs for each step of many requests at once (no counterpart in the
 * reference, whose KvCache holds one request in fp32). Like the QuantMatMul section they take
 * device pointers and a cudaStream_t and return once the work is queued; they allocate nothing,
 * so a step can be captured in a CUDA graph and replayed with other lengths. Each runs on the
 * device that its buffers are on, whichever is current; `stream` must belong to that device.
 * Calls that write the same cache pages, batch arrays or workspace must be ordered by the
 * caller (one stream, or events): two graphs that share them must not run at the same time.
 * What only the device knows (lengths, page ids, slots) is checked there: a bad value is not
 * used but recorded in the two-word status (word 0 a JV_* status, the first one stays; word 1
 * the site), which the caller zeroes once and reads when it likes.
 *
 * type is a GGML type id: 0 F32, 1 F16, 30 BF16. */

#define JV_PAGE_TOKENS 64  /* tokens per page                                   */
#define JV_SCALE_TOKENS 16 /* tokens that share a scale, per KV head and K or V */

/* One layer of the cache. Page p holds int8 [kv_heads][2 (K, V)][64][128] at data + p * page_bytes
 * (bytes; at least kv_heads * 16384, a multiple of 16) and fp32 [kv_heads][2][4], one scale for each
 * 16 tokens, at scales + p * scale_stride (floats; at least kv_heads * 8, a multiple of 4): the value
 * is int8 * scale. data and scales are 16-byte aligned. Layers may be interleaved inside a page
 * through the strides. head_dim is 128. */
typedef struct jv_kv8_cache {
    void* data;
    float* scales;
    int64_t page_bytes, scale_stride;
    int32_t pages, kv_heads;
} jv_kv8_cache;

/* A step of `requests` requests (1..4096) and the arrays jv_paged_plan writes for it. The bounds
 * are the caller's; a step beyond one of them fails as a whole. group is the number of query heads
 * per KV head (1..16). Rows of the token arrays behind the step's last token are left as they were. */
typedef struct jv_paged_batch {
    int32_t requests;
    int32_t max_new;      /* most new tokens of one request                                */
    int32_t max_tokens;   /* most new tokens of all requests: rows of the token arrays     */
    int32_t max_blocks;   /* most pages of one request: columns of block_table             */
    int64_t max_keys;     /* most tokens of all requests after the step                    */
    int32_t group;        /* query heads per KV head                                       */
    int32_t pages;        /* pages of the cache                                            */
    int32_t* block_table; /* [requests][max_blocks] page of tokens 64 b .. 64 b + 63; in, out */
    int32_t* lengths;     /* [requests] tokens after the step                              */
    int32_t* starts;      /* [requests + 1] first new token of each request; the last: all */
    int32_t* request_of;  /* [max_tokens]                                                  */
    int32_t* positions;   /* [max_tokens]                                                  */
    int64_t* slots;       /* [max_tokens] page * 64 + position % 64                        */
    void* work;           /* jv_paged_work_bytes bytes, 16-byte aligned                    */
    int32_t* status;      /* [2]                                                           */
} jv_paged_batch;

/* Bytes of jv_paged_batch.work for the batch's bounds; -1 and jv_last_error on a bad one, or where they allow
 * 2^30 chunks of work (64 to 2048 keys of 16 query rows) or more, which every operator refuses. */
int64_t jv_paged_work_bytes(const jv_paged_batch* batch);

/* Block tables and slot maps from the requests' lengths. Request r holds cached[r] tokens, whose
 * pages are in its row of block_table, and brings new_tokens[r] (0 allowed). The pages it lacks are
 * taken from the end of free_pages[*n_free] (in request order, then block order: free_pages[*n_free
 * - 1] first) and *n_free_out becomes the count left. Every array of the batch is written. cached may
 * be lengths and n_free_out may be n_free, for a step that continues the last. Requests may share
 * pages that are full; a page that a request writes to must be its own, and free_pages must not name a
 * page twice or one in use.
 * If a bound of the batch is exceeded (JV_ERR_RANGE), free pages run out (JV_ERR_OOM) or a free page
 * is not in the cache (JV_ERR_RANGE), no page is taken, lengths become cached and starts 0: the
 * operators after it then do nothing. */
int jv_paged_plan(const jv_paged_batch* batch, const int32_t* cached, const int32_t* new_tokens, const int32_t* free_pages,
                  const int32_t* n_free, int32_t* n_free_out, void* stream);

enum jv_rope_layout { JV_ROPE_ADJACENT = 0 /* pairs (2i, 2i + 1) */, JV_ROPE_HALF = 1 /* pairs (i, i + rotary_dim / 2) */ };
enum jv_rope_scaling { JV_ROPE_PLAIN = 0, JV_ROPE_LINEAR = 1, JV_ROPE_YARN = 2 };

/* Rotary positions (the rule of src/Jevstral/Model/Rope.cs:33-106, with angles in 64 bits, so that far
 * positions keep theirs). turns[i] is pair i's frequency in turns per position; mscale multiplies every
 * rotated element. temperature_scale and temperature_ctx are the query temperature of
 * MinistralModel.cs:676-682 (off when either is 0): 1 + scale * ln(1 + floor(position / ctx)) on every
 * element of heads that ask for it. jv_rope_init fills the struct; it is passed by value to the kernels. */
typedef struct jv_rope_spec {
    int32_t layout, rotary_dim;
    float mscale, temperature_scale;
    int32_t temperature_ctx, reserved;
    double turns[128];
} jv_rope_spec;

/* rotary_dim: even, 2..256. factor > 0 (used by LINEAR and YARN), original_context, beta_fast and
 * beta_slow (YARN). mscale is attn_factor, times 0.1 ln(factor) + 1 for YARN with factor > 1. */
int jv_rope_init(jv_rope_spec* out, int32_t layout, int32_t rotary_dim, double base, int32_t scaling, double factor,
                 int32_t original_context, double beta_fast, double beta_slow, double attn_factor);

/* [tokens][heads][dim] in device memory, the last dimension contiguous; strides in elements. out may
 * be NULL where only `in` is used, and may be `in` (with the same strides) for an operator in place;
 * in and out must not overlap in any other way. */
typedef struct jv_heads {
    const void* in;
    void* out;
    int64_t in_token, in_head, out_token, out_head;
    int32_t heads;
    int32_t temperature; /* apply the spec's query temperature */
} jv_heads;

/* Rotates x[0..n) (queries and keys, n = 1 or 2) at positions[tokens]; the elements from rotary_dim on
 * are copied. head_dim: even, up to 256, at least rotary_dim. tokens == 0 does nothing. A result outside
 * the type's range becomes an infinity. */
int jv_rope(const jv_rope_spec* spec, int32_t type, const int32_t* positions, int32_t tokens, int32_t head_dim,
            const jv_heads* x, int32_t n, void* stream);

/* Writes the batch's new keys and values (k->in and v->in, [tokens][kv_heads][128]) to their slots in 8
 * bits. A block of 16 tokens has one scale per head for K and one for V: the largest magnitude written
 * to it / 127. Where a block holds tokens of earlier steps the scale grows if it must, and their entries
 * are rounded again at the new scale. With `rope` the keys are rotated first (rotary_dim a multiple of 8,
 * at most 128) and, with q, the queries too: q->in of `type` to q->out of out_type. Only q may ask for the
 * query temperature. A value that is not finite is recorded as JV_ERR_NUMERIC; it is stored as 0 (not a
 * number) or the block's largest value (an infinity) and does not count for the scale. Magnitudes below
 * 2^-100 are stored as 0. */
int jv_kv8_append(const jv_kv8_cache* cache, const jv_paged_batch* batch, int32_t type, const jv_heads* k,
                  const jv_heads* v, const jv_rope_spec* rope, const jv_heads* q, int32_t out_type, void* stream);

/* The values at slots[n] (page * 64 + row): k_out and v_out, [n][kv_heads][128] of `type`, rows
 * `row_stride` elements apart. The rows of a negative slot are left as they were; a slot past the
 * cache is recorded as JV_ERR_RANGE and its rows are left too. status may be NULL. */
int jv_kv8_read(const jv_kv8_cache* cache, const int64_t* slots, int32_t n, int32_t type, void* k_out, void* v_out,
                int64_t row_stride, int32_t* status, void* stream);

/* Bytes of the workspace of jv_kv8_attention for the batch's bounds (nothing in it has to be
 * initialised, and nothing is kept in it); -1 on a bad batch. */
int64_t jv_kv8_attention_bytes(const jv_paged_batch* batch, int32_t kv_heads);

/* Grouped-query attention of the batch's new tokens over the cache (their own keys appended before):
 * q->in, [tokens][kv_heads * group][128] of `type` (F16 or BF16), to q->out of the same type. The token
 * at position p sees keys p - window + 1 .. p, or 0 .. p when window is 0. A token without a visible key
 * gives zeros; the keys of a page that is not in the cache (recorded as JV_ERR_RANGE) have no weight. An
 * F16 output outside the type's range becomes an infinity; that, and an F16 output that is not a number, is
 * recorded as JV_ERR_NUMERIC. The result of a request depends on its own tokens only, bit for bit, not on
 * what else is in the batch or on its bounds. Rows of q start on 16 bytes.
 * Scores, exponents, sums and the softmax's denominator are fp32; a weight is rounded to fp16 before it meets
 * the values, by half a step (2^-11 of itself, or 2^-25 of the row's largest product of weight and block scale
 * where that is more). That holds for values of 2^-50 to 2^40 where blocks of zeros are beside them, and for
 * |scale * q| up to 2^110. */
int jv_kv8_attention(const jv_kv8_cache* cache, const jv_paged_batch* batch, int32_t type, const jv_heads* q, float scale,
                     int32_t window, void* workspace, int64_t workspace_bytes, void* stream);

/* ---- many requests of one model, stepped together (no counterpart in the reference) ------
 * A jv_server holds an 8-bit KV cache (the paged-batch section above: half the bytes per position
 * of a context's fp16 pages) for up to max_requests requests, and runs the new tokens of any of
 * them in one pass: one product per weight matrix for all, plan, rotation and append, attention,
 * and the head's rows at each request's last token. Like a jv_ctx it is single-threaded, and it
 * shares the jv_model's weights. A request's results do not depend, bit for bit, on what else is in
 * the pass. */

/* max_context: most positions of a request; max_tokens: most new tokens of one pass; pages: pages of
 * 64 positions shared by the requests (0 = max_context positions for every request). Beside the pages the
 * server holds a quarter of a page for each request that a pass can continue (at most max_requests,
 * max_tokens and pages), to put back what a failed pass changed. */
int jv_server_create(jv_model* model, int32_t max_requests, int32_t max_context, int32_t max_tokens, int32_t pages,
                     jv_server** out);
void jv_server_destroy(jv_server* server);
/* One pass: request r brings counts[r] tokens (0: it sits the pass out), back to back in `tokens` in
 * request order. out[requests with tokens][n_rows] = logits of vocabulary `rows` at each one's last
 * token, in request order. A pass that fails leaves every request as it was: JV_ERR_OOM when the pages
 * run out, JV_ERR_RANGE when a request would pass max_context, and errors found on the device
 * (JV_ERR_NUMERIC; the blocks of 16 positions that the pass continued are put back). */
int jv_server_forward(jv_server* server, const int32_t* tokens, const int32_t* counts, const int32_t* rows,
                      int32_t n_rows, float* out);
/* Ends a request: its positions go to 0 and its pages back to the others. */
int jv_server_release(jv_server* server, int32_t request);
int32_t jv_server_length(const jv_server* server, int32_t request); /* positions held; -1 for a bad index */
int64_t jv_server_bytes_per_position(const jv_server* server);

/* ---- KV cache (src/Jevstral/Model/KvCache.cs) ----------------------------------------- */

int32_t jv_kv_length(jv_ctx* ctx);                             /* KvCache.Length   :23     */
int32_t jv_kv_capacity(jv_ctx* ctx);                           /* KvCache.Capacity :21     */
int jv_kv_reset(jv_ctx* ctx);                                  /* KvCache.Reset    :43     */
int jv_kv_truncate(jv_ctx* ctx, int32_t length);               /* KvCache.Truncate :46     */
int jv_kv_ensure_capacity(jv_ctx* ctx, int32_t required);      /* EnsureCapacity   :48-70  */
int64_t jv_kv_bytes_per_position(jv_ctx* ctx);                 /* BytesPerPosition :139    */
/* KvCache.Snapshot (:94-112): the reference's flat fp32 layout (keys for every layer and
 * head, then values), so SystemPromptCache files (SystemPromptCache.cs:110-164) stay valid.
 * n_floats must equal jv_kv_snapshot_floats(length). */
int64_t jv_kv_snapshot_floats(jv_ctx* ctx, int32_t length);
int jv_kv_snapshot(jv_ctx* ctx, int32_t length, float* out, int64_t n_floats);
/* KvCache.Restore (:115-136). */
int jv_kv_restore(jv_ctx* ctx, const float* snapshot, int64_t n_floats, int32_t length);

/* SystemPromptCache.Save (src/Jevstral/SystemPromptCache.cs:110-127) straight from the device
 * pages: writes the reference's "SHKV" file for the first n_tokens cached positions — uint32
 * magic 0x53484B56, int32 version 1, the fingerprint string as .NET's BinaryWriter writes it
 * (7-bit-encoded UTF-8 byte count, then the bytes), int32 token count, the tokens, int64 float
 * count, then the KvCache.Snapshot floats (:94-112) — streamed one (K|V, layer) slice at a time
 * through pinned memory, so the whole state never sits in host memory. The fingerprint is the
 * host's (ComputeFingerprint, :91-106); n_tokens must not exceed the cached length. */
int jv_kv_save_shkv(jv_ctx* ctx, const char* path, const char* fingerprint, const int32_t* tokens, int32_t n_tokens);
/* SystemPromptCache.TryLoad + RestoreInto (SystemPromptCache.cs:65-74,133-164) into the device
 * pages: reads an SHKV file, checks its magic, version, that its fingerprint equals `fingerprint`
 * and that its float count fits its token count on this model, then streams the floats into the
 * pages (the cache then holds exactly that prefix) and writes the tokens to tokens_out
 * (max_tokens entries) and their count to *n_tokens. TryLoad's miss (null) is JV_ERR_IO for a file
 * that cannot be opened and JV_ERR_FORMAT for one that is not a valid snapshot of this model and
 * prefix; both leave the cache as it was. */
int jv_kv_load_shkv(jv_ctx* ctx, const char* path, const char* fingerprint, int32_t* tokens_out, int32_t max_tokens,
                    int32_t* n_tokens);

/* Zero-copy prefix reuse (the question-snapshot LRU and system-prompt cache of
 * JevstralDecider.cs:131-137,262-280 without the memcpy): jv_kv_share pins the pages that
 * hold the first `length` positions; jv_kv_adopt makes a context's cache exactly that prefix
 * (copy-on-write for the one partially filled page). Contexts must share the jv_model. */
int jv_kv_share(jv_ctx* ctx, int32_t length, jv_snapshot** out);
int jv_kv_adopt(jv_ctx* ctx, const jv_snapshot* snapshot);
int32_t jv_snapshot_length(const jv_snapshot* snapshot);
void jv_snapshot_release(jv_snapshot* snapshot);

#ifdef __cplusplus
}
#endif

#endif /* JV_H */
