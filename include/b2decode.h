/*
 * b2decode — B200 (sm_100a) decode engine for GGUF Q8_0 / Q4_0 LLaMA/Qwen2
 * models, a drop-in for the per-token forward pass of the Local-LLM-Pure-Go
 * engine.
 *
 * C ABI: plain pointers and sizes, no C++ or CUDA types.  Every function that
 * can fail returns 0 on success or a negative B2_ERR_* code; the message of
 * the last failure on the calling thread is b2_last_error().  No exception or
 * abort crosses the ABI.  The library owns all device memory of a model.  Host
 * buffers passed in are read or written only during the call.  Calls on one
 * b2_model must be serialised by the caller (the Go engine holds one
 * sync.Mutex per engine, transformer.go:96).
 *
 * Reference interfaces replaced (paths relative to the reference project):
 *   Local-LLM-Pure-Go/internal/engine/engine.go:15-39          Engine interface
 *   Local-LLM-Pure-Go/internal/engine/native/transformer/transformer.go
 *   Local-LLM-Pure-Go/internal/engine/native/gguf/gguf.go
 */
#ifndef B2DECODE_H
#define B2DECODE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B2_OK 0
#define B2_ERR_IO (-1)               /* file missing or short read */
#define B2_ERR_FORMAT (-2)           /* bad magic/version, truncated or inconsistent GGUF */
#define B2_ERR_UNSUPPORTED_TYPE (-3) /* tensor type the engine cannot run */
#define B2_ERR_OOM (-4)              /* device or host allocation failed */
#define B2_ERR_CUDA (-5)             /* CUDA runtime error */
#define B2_ERR_NCCL (-6)             /* collective failure */
#define B2_ERR_TIMEOUT (-7)          /* a bounded device-side wait gave up */
#define B2_ERR_BAD_ARG (-8)          /* invalid argument */
#define B2_ERR_CONTEXT (-9)          /* position beyond the KV-cache capacity */
#define B2_ERR_NOT_LOADED (-10)      /* model handle is NULL or unloaded */

typedef struct b2_model b2_model;
typedef struct b2_batch b2_batch;

/* engine.go:42-47 LoadOptions, plus device placement. */
typedef struct {
    int32_t num_ctx;    /* LoadOptions.NumCtx: caps context_length when > 0 (transformer.go:233-235) */
    int32_t device;     /* CUDA device ordinal */
    int32_t kv_fp32;    /* 0: fp16 KV cache (default); 1: fp32 KV cache as in the Go engine */
    int32_t tp_size;    /* LoadOptions.NumGPU: tensor-parallel degree (0 or 1: one GPU; up to 8) */
    int32_t tp_rank;    /* this process's rank, 0 .. tp_size - 1 (one process per GPU) */
    int32_t reserved2;
} b2_load_opts;

/* transformer.go:33-46 ModelConfig, plus what loadWeights derives. */
typedef struct {
    char arch[32];
    int32_t vocab_size;
    int32_t hidden_size;
    int32_t intermediate_size;
    int32_t num_layers;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t head_dim;
    int32_t max_seq_len;       /* min(context_length, num_ctx) */
    float rms_norm_eps;
    float rope_theta;
    int32_t tied_embeddings;   /* 1: lm_head reads token_embd (transformer.go:551-554) */
    int32_t has_qkv_bias;
    int32_t weight_type;       /* ggml type of the layer matrices: 8 = Q8_0, 2 = Q4_0 */
    int32_t bos_id;            /* tokenizer.ggml.bos_token_id (bpe.go:48,105) */
    int32_t eos_id;            /* tokenizer.ggml.eos_token_id (bpe.go:49,108) */
    int64_t weight_bytes;      /* bytes of weights resident in HBM (this rank's) */
    int64_t stream_bytes_per_token; /* algorithmic HBM bytes one B=1 decode token reads (this rank's) */
    int32_t tp_size;           /* tensor-parallel degree and this rank */
    int32_t tp_rank;
    int32_t vocab_begin;       /* this rank's share of the lm_head rows: logits of */
    int32_t vocab_local;       /* vocab ids vocab_begin .. vocab_begin + vocab_local - 1 */
} b2_config;

/* Real phase timings (the Go engine reports fixed 1/3 and 2/3 splits,
 * transformer.go:379-380). */
typedef struct {
    int64_t prompt_ns;
    int64_t eval_ns;
    int32_t prompt_tokens;
    int32_t completion_tokens;
} b2_timings;

/* domain.Options (internal/domain/types.go:142-160) fields used by sample. */
typedef struct {
    double temperature;     /* <= 0 means 1.0; greedy when < 0.01 (transformer.go:982-1004) */
    int32_t top_k;
    double top_p;
    double repeat_penalty;  /* applied when > 1 */
    int32_t num_predict;    /* <= 0 means 256 */
    uint64_t seed;          /* seed of the engine's uniform generator */
} b2_sample_opts;

/* ---- model lifecycle (engine.go Load/Unload/ModelInfo/IsLoaded) ---- */

/* transformer.go:215-310 Engine.Load: parse the GGUF, extract the config,
 * copy every Q8_0/Q4_0 block verbatim into one HBM arena (no host dequant),
 * allocate the KV cache.  opts may be NULL. */
int b2_load(const char* gguf_path, const b2_load_opts* opts, b2_model** out);
/* transformer.go:312-322 Unload. NULL is ignored. */
void b2_free(b2_model* m);
int b2_get_config(const b2_model* m, b2_config* out);

/* Where b2_load's time went (transformer.go:1122-1335 loadWeights reads and
 * dequantises on the host; here the blocks go to HBM as they are): the file
 * is memory-mapped, a pool of host threads copies each 32 MB range into one
 * of four pinned stages while the previous stages' cudaMemcpyAsync run, and
 * the device retiles each matrix. */
typedef struct {
    int64_t total_ns;        /* the whole b2_load */
    int64_t parse_ns;        /* GGUF header, metadata and tensor infos */
    int64_t upload_ns;       /* weight and vector bytes to HBM, retiling included */
    int64_t host_copy_ns;    /* of upload_ns: host threads filling the pinned stages */
    int64_t bytes_uploaded;  /* weight bytes sent through the stages */
    int32_t host_threads;
    int32_t mapped;          /* 1: memory-mapped file; 0: pread */
    int64_t setup_ns;        /* of upload_ns: mapping the file, pinned stages, thread pool */
} b2_load_stats;
int b2_get_load_stats(const b2_model* m, b2_load_stats* out);
/* Message of the last failure on this thread ("" if none). */
const char* b2_last_error(void);

/* ---- forward pass ---- */

/* transformer.go:742-749 resetCache. */
int b2_reset(b2_model* m);
/* Number of cached positions (kvCache.Len, transformer.go:88-92). */
int b2_cache_len(const b2_model* m, int32_t* len_out);

/* transformer.go:519-557 forward: run n tokens (prefill when n > 1) from the
 * current cache position; write the vocab_size logits of the last token to
 * logits_out (may be NULL). */
int b2_forward(b2_model* m, const int32_t* tokens, int32_t n, float* logits_out);
/* forward followed by argmax (transformer.go:1038-1046, first maximum wins)
 * computed on the device. */
int b2_forward_argmax(b2_model* m, const int32_t* tokens, int32_t n, int32_t* next_out);
/* Device-resident greedy loop: feed `first`, then each argmax, n_steps times;
 * stop after emitting eos (eos < 0 disables the stop).  out_ids receives up to
 * n_steps ids, *n_out how many (the eos id itself is not emitted, as in
 * Predict, transformer.go:355-357). */
int b2_decode_greedy(b2_model* m, int32_t first, int32_t n_steps, int32_t eos, int32_t* out_ids,
                     int32_t* n_out);

/* ---- engine loop (engine.go Predict / PredictStream on token ids) ---- */

/* transformer.go:325-382 Predict: reset, prepend BOS, prefill, then up to
 * num_predict steps of forward + sample, stopping at EOS or at any id in
 * stop_ids (the token-id form of isStopToken, transformer.go:1430-1437).
 * Greedy runs device-resident; otherwise each step's logits are sampled on
 * the device by the b2_sample_device sampler (transformer.go:981-1114), with
 * the engine's seeded uniforms, and only the id comes back. */
int b2_predict(b2_model* m, const int32_t* prompt, int32_t n_prompt, const b2_sample_opts* opts,
               const int32_t* stop_ids, int32_t n_stop, int32_t* out_ids, int32_t max_out, int32_t* n_out,
               b2_timings* timings);
/* transformer.go:385-442 PredictStream as an iterator: begin resets and
 * prefills; each next call yields one token id or done=1 (EOS, stop id or
 * num_predict reached). */
int b2_stream_begin(b2_model* m, const int32_t* prompt, int32_t n_prompt, const b2_sample_opts* opts,
                    const int32_t* stop_ids, int32_t n_stop);
int b2_stream_next(b2_model* m, int32_t* token_out, int32_t* done_out);

/* transformer.go:981-1036 sample() on host logits (modified in place), with
 * the caller's uniform r in [0,1) for the multinomial draw. */
int32_t b2_sample_logits(float* logits, int32_t n, const b2_sample_opts* opts, const int32_t* generated,
                         int32_t n_generated, float r);
/* transformer.go:981-1114 sample() on the DEVICE, the sampler b2_predict and
 * b2_stream_next use: rows (<= 64) sequences, row i's logits at
 * d_logits[i * ld .. + n) in device memory (modified in place: penalty,
 * temperature, filtered entries), its generated ids at d_generated[i * gen_ld
 * .. + n_generated[i]) (device; may be NULL without a penalty), its uniform
 * r[i] in [0,1) (host array).  Top-K and top-P are radix selections (no
 * sort) by a group of CTAs per row; the masses are summed exactly in fixed
 * point, so the id equals the host sampler's except where r or top_p lies
 * within the host's float rounding of a cumulative boundary.  d_scratch:
 * b2_sample_scratch_bytes(n, rows) bytes of device memory.  The ids are
 * written to d_out[rows] (device; -1 if a group barrier of the launch ran
 * out); asynchronous on stream (a cudaStream_t; NULL = the legacy default
 * stream). */
int64_t b2_sample_scratch_bytes(int32_t n, int32_t rows);
int b2_sample_device(float* d_logits, int32_t n, int32_t rows, int64_t ld, const b2_sample_opts* opts,
                     const int32_t* d_generated, int64_t gen_ld, const int32_t* n_generated, const float* r,
                     void* d_scratch, int32_t* d_out, void* stream);

/* transformer.go:445-490 Embed: mean of the token_embd rows of the ids,
 * L2-normalised, written to out[hidden_size]. */
int b2_embed(b2_model* m, const int32_t* tokens, int32_t n, float* out);

/* ---- debug / kernel-level entry points ---- */

/* gguf.go:491-508 Dequantize of one named tensor, decoded on the device from
 * the resident blocks (Q4_0 in the ggml element order).  n = capacity of out
 * in floats; returns 0 and writes *n_out elements.  On a tensor-parallel rank
 * a sharded tensor yields this rank's share (its rows, or its columns of each
 * row, in the order of the GGUF tensor). */
int b2_dequant_tensor(const b2_model* m, const char* name, float* out, int64_t n, int64_t* n_out);

/* transformer.go:810-865 matVecMulQ8Chunk over all rows, on the device:
 * y[r] = sum_b d_b * sum_j q_bj * x[32b+j].  w, x, y are DEVICE pointers
 * (GGUF block rows, fp32).  qtype 8 = Q8_0, 2 = Q4_0 (ggml layout).
 * stream is a cudaStream_t (NULL = legacy default stream). */
int b2_matvec(int32_t qtype, const void* w, const float* x, float* y, int32_t rows, int32_t cols,
              void* stream);

/* transformer.go:810-892 (matVecMulQ8Chunk / matVecMulQ8Pooled) for nvec
 * vectors at once, reading the matrix from HBM once: y[v][r] = sum_b d_rb *
 * sum_j q_rbj * x[v][32b+j] for v < nvec.  x [nvec][cols] and y [nvec][rows]
 * fp32, w GGUF block rows (16-byte aligned); all DEVICE pointers.
 * 1 <= nvec <= 16 (vectors 8..15 share the pass over w with 0..7); cols a
 * multiple of 256.  qtype 8 = Q8_0, 2 = Q4_0.  Uses a
 * scratch buffer per (device, stream), grown with cudaMalloc when a call
 * needs more; calls on one stream run in order, calls on different streams
 * use different buffers. */
int b2_matvec_batch(int32_t qtype, const void* w, const float* x, float* y, int32_t rows, int32_t cols,
                    int32_t nvec, void* stream);
/* The same batched dots (transformer.go:810-892 for nvec vectors) over a
 * weight matrix of the loaded model, read from its resident tiled blocks:
 * y[v][r] = sum_j W[r][j] * x[v][j] for the tensor `name` (this rank's share
 * under tensor parallelism, rows and columns as b2_dequant_tensor returns
 * them).  x [nvec][cols], y [nvec][rows] fp32 DEVICE pointers, 1 <= nvec <=
 * 16; the model's device must be current.  stream NULL = the model's own
 * stream.  The gate and up matrices are stored interleaved and are rejected.
 * Shares the per-(device, stream) scratch of b2_matvec_batch. */
int b2_model_matvec(const b2_model* m, const char* name, const float* x, float* y, int32_t nvec, void* stream);
/* The same product for any number of tokens on the tensor cores (tcgen05,
 * TMA-staged tiles): Y = W X for the tensor `name`, x [ntok][cols], y
 * [ntok][rows] fp32 DEVICE pointers, ntok >= 1, cols a multiple of 64.  The
 * weights are decoded to fp16 in shared memory (d * q rounded once) and the
 * activations converted to fp16 with a power-of-two scale per token; products
 * accumulate in fp32.  This is the dense contraction of a prompt's prefill:
 * the batched counterpart of the C++ sibling engine's
 * Local-LLM/include/tensor.h:354-387 mat_mat_mul_tensor (Transformer::
 * forward_batch, Local-LLM/src/transformer.cpp:540-575).  Asynchronous on
 * `stream` (NULL = the model's stream), with a per-(device, stream) scratch
 * grown by cudaMalloc when a call needs more.  The gate and up matrices,
 * stored interleaved, are computed whole and their half gathered (a buffer
 * of ntok x 2 x rows floats allocated on the stream for the call). */
int b2_model_gemm(const b2_model* m, const char* name, const float* x, float* y, int32_t ntok, void* stream);

/* transformer.go:663-685 attention of one query token per sequence over an
 * fp16 KV cache, split over the context with a log-sum-exp merge.
 * q [batch][nh*hd] fp32; k, v [batch][ctx][nkv*hd] fp16 (binary16 bits);
 * out [batch][nh*hd] fp32.  DEVICE pointers.  Asynchronous on `stream`; the
 * split partials live in a scratch kept per (device, stream), grown by
 * cudaMalloc when a call needs more and held until the process exits, so
 * calls on different streams may overlap (a caller that cycles through many
 * short-lived streams holds one buffer per stream it used). */
int b2_attention_decode(const float* q, const uint16_t* k, const uint16_t* v, float* out, int32_t batch,
                        int32_t nh, int32_t nkv, int32_t hd, int32_t ctx, void* stream);

/* b2_attention_decode without any device allocation, for callers that cannot
 * call cudaMalloc: a serving process whose HBM is already fully reserved by
 * its own pools (weights, KV cache), or a per-token path that cannot afford
 * the device-wide synchronisation a cudaMalloc/cudaFree pair can cause.  The
 * split partials use a fixed 2 MiB device array inside the library (held by
 * every GPU that loads it until the process exits); the caller still passes
 * q, k, v and out.  Limit: batch * nh * (hd + 2) <= 524288 floats, larger
 * sizes fail with B2_ERR_BAD_ARG.  The first call on a device looks up the
 * array's device address; make that first call before any stream capture.
 * The address is cached per device for the life of the process: after a
 * caller resets a device (cudaDeviceReset) this entry point must not be
 * called on it again.  All calls share the array, so calls whose kernels
 * overlap on the GPU race.  No counterpart in the reference. */
int b2_attention_decode_noalloc(const float* q, const uint16_t* k, const uint16_t* v, float* out, int32_t batch,
                                int32_t nh, int32_t nkv, int32_t hd, int32_t ctx, void* stream);

/* ---- batched greedy decode (config: Llama-3-8B at batch 16) ----
 *
 * Up to 16 sequences, each with a KV-cache slot of its own (max_seq = the
 * model's num_ctx, fp16), advance one token per b2_batch_step together, each
 * at its own position, so every weight byte is read once per step for all of
 * them: the forward of transformer.go:519-739 and argmax 1038-1046 for B
 * sequences at a time.  b2_batch_prefill runs a slot's prompt into the slot
 * (the model's own single-sequence cache is not touched); next_out is the
 * argmax after the prompt.  b2_batch_step
 * feeds tokens[B] (one per slot, every slot) and writes the B argmax ids;
 * b2_batch_logits copies the logits of the last forward of the batch,
 * [B][vocab_size]: the B rows of the last b2_batch_step, or, after a
 * b2_batch_prefill, the prompt's last token in row 0.  A prompt runs in
 * chunks of up to 256 of its tokens, each one pass over the weights on the
 * tensor cores (b2_model_gemm's product) with the chunk's attention over the
 * slot's cache.  Needs a
 * single-GPU model with the fp16 cache; the model's device must be current.
 * Every batch of a model runs on the model's stream and shares its scratch,
 * so calls on the batches of one model, like calls on the model itself, must
 * be serialised by the caller; batches of different models are independent.
 * A batch is used only while its model is loaded; b2_batch_free may come
 * before or after b2_free of the model.
 * No single counterpart in the reference (its engine runs one sequence). */
int b2_batch_create(b2_model* m, int32_t batch, b2_batch** out);
void b2_batch_free(b2_batch* b);
int b2_batch_prefill(b2_batch* b, int32_t slot, const int32_t* prompt, int32_t n, int32_t* next_out);
int b2_batch_step(b2_batch* b, const int32_t* tokens, int32_t* next_out);
int b2_batch_logits(const b2_batch* b, float* out);
/* b2_logprobs on those logits where they are, in device memory: rows (at most
 * the batch after a b2_batch_step, 1 after a b2_batch_prefill; more, or any
 * without a forward before, fail with B2_ERR_BAD_ARG) rows, ids [rows][m] and the results
 * ([rows][m], [rows], [rows][k] twice) in HOST memory, entropy may be NULL.
 * Returns when the results are there.  The Go engine returns no scores. */
int b2_batch_logprobs(const b2_batch* b, int32_t rows, const int32_t* ids, int32_t m, float* logprob, float* entropy,
                      int32_t k, int32_t* top_ids, float* top_logprob);
/* on != 0: replay each step's launches from a CUDA graph, captured after the
 * first step that runs with the switch on (and again after the batched
 * matvec's shared scratch has moved); a capture that fails leaves the batch
 * stepping eagerly.  Off by default. */
int b2_batch_use_graph(b2_batch* b, int32_t on);

/* ---- paged serving step: plan, rotate + append, attend, score ----
 *
 * A server that keeps its KV cache in pages (blocks of page_size positions,
 * handed out as sequences grow) runs a step in this order: b2_page_plan takes
 * pages from the free list and says where every token of the step goes;
 * b2_rope_append rotates q and k and writes k and v to those places;
 * b2_attention_paged attends, one query row per token; b2_logprobs scores the
 * logits.  Kernel-level entry points: DEVICE pointers unless said otherwise,
 * on the current device (host memory, or another device's, fails with
 * B2_ERR_BAD_ARG), asynchronous on `stream` (a cudaStream_t; NULL = the legacy
 * default stream), no allocation, no state kept between calls, capturable in a
 * CUDA graph.  Calls that overlap on the GPU must not share outputs or
 * scratch.  An output shares no memory with an input or another output, unless
 * its entry point says that it may.  Types are ggml type ids: 0 = F32, 1 = F16, 30 = BF16.  The Go
 * engine has one contiguous cache per sequence (kvCache,
 * transformer.go:88-92); these have no counterpart there beyond the
 * arithmetic cited. */

/* A paged KV cache: the element d of head h of position s of page p is at
 * k[p * page_stride + s * pos_stride + h * head_stride + d], v alike.  Strides
 * in elements; all three 0 = dense [n_pages][page_size][nkv][hd].  k and v on
 * 16 bytes, strides multiples of 8, hd a multiple of 8 up to 256. */
typedef struct {
    void* k;
    void* v;
    int32_t dtype; /* 1 = F16, 30 = BF16 */
    int32_t n_pages;
    int32_t page_size;
    int32_t nkv;
    int32_t hd;
    int32_t reserved;
    int64_t page_stride;
    int64_t pos_stride;
    int64_t head_stride;
} b2_paged_kv;

/* Why a plan did not fit: bits of b2_page_plan's info[0]. */
#define B2_PLAN_BAD_LENGTH 1 /* a negative length */
#define B2_PLAN_TABLE_FULL 2 /* a request needs more than max_pages pages, or passes 2^31 - 1 positions */
#define B2_PLAN_ROWS_FULL 4  /* more new tokens than max_tokens */
#define B2_PLAN_NO_PAGES 8   /* more new pages than *n_free */

/* Block tables and slot maps from request lengths.  Request r (of n_req, at
 * most 16384) holds cached[r] positions in the first ceil(cached[r] /
 * page_size) entries of its table row (table + r * table_stride, max_pages
 * entries) and gets fresh[r] >= 0 more tokens.  New pages are taken from the
 * front of free_pages (*n_free of them, a device word), in request order.
 * Writes
 *   table      the new entries, nothing else
 *   lens[r]    cached[r] + fresh[r]
 *   starts     [n_req + 1] first token row of each request, and the total
 *   slots, positions, token_req  [max_tokens], for each token in request
 *              order: page * page_size + place in the page, the position, the
 *              request; the rows past the last token get -1, 0, -1
 *   info       [4] {status, tokens, pages taken, 0}
 * A step that does not fit (status != 0, B2_PLAN_* bits) leaves the table as
 * it was and is an empty one otherwise: every token row -1, starts 0, lens =
 * cached.  A token in a page whose table or list entry is negative gets slot
 * -1.  No two requests may share a page that either still writes.  The outputs
 * and the table share no memory with cached, fresh, n_free, free_pages or one
 * another (the lengths are read again while others are written, so lens is no
 * update of cached in place): a call whose output meets an input or the table
 * fails with B2_ERR_BAD_ARG, for free_pages as far as its first entry, its
 * length being on the device. */
int b2_page_plan(const int32_t* cached, const int32_t* fresh, int32_t n_req, int32_t page_size,
                 const int32_t* free_pages, const int32_t* n_free, int32_t* table, int64_t table_stride,
                 int32_t max_pages, int32_t* lens, int32_t* starts, int64_t* slots, int32_t* positions,
                 int32_t* token_req, int32_t max_tokens, int32_t* info, void* stream);

#define B2_ROPE_INTERLEAVED 0 /* pairs (2i, 2i + 1), as transformer.go:936-951 rotates */
#define B2_ROPE_HALF 1        /* pairs (i, i + rot_dim / 2) */

#define B2_ROPE_SCALE_NONE 0
#define B2_ROPE_SCALE_LINEAR 1 /* every frequency over factor */
#define B2_ROPE_SCALE_BANDS 2  /* over factor where a pair turns at most `low` times in orig_ctx positions, kept
                                  where it turns at least `high` times, blended linearly in the turns between */
#define B2_ROPE_SCALE_YARN 3   /* the same ends, blended linearly in the pair's number; cos and sin times
                                  0.1 log(factor) + 1 */

typedef struct {
    int32_t rot_dim; /* rotated elements of a head (even) */
    int32_t scaling; /* B2_ROPE_SCALE_* */
    double theta;    /* rope_theta, > 1 */
    double factor;   /* context stretch, > 0 (ignored for NONE) */
    double orig_ctx; /* positions the model was trained on, > 0 (BANDS, YARN) */
    double low;      /* <= 0: 1 */
    double high;     /* <= 0: 4 (BANDS) or 32 (YARN) */
} b2_rope_opts;

/* The frequencies of b2_rope, radians per position, freqs[rot_dim / 2] (HOST
 * memory; a server uploads them once), and the factor on cos and sin (scale;
 * may be NULL).  transformer.go:939-942 is theta^(-2i/hd), in float64. */
int b2_rope_freqs(const b2_rope_opts* opts, double* freqs, float* scale);

/* The rows of a step: q [n_tok] rows of nh heads, k and v [n_tok] rows of nkv
 * heads, hd elements a head (even, at most 256), heads back to back in a row.
 * Strides in elements from row to row; 0 = dense.  Any alignment; rows on 16
 * bytes run fastest. */
typedef struct {
    int32_t dtype; /* q, k, v, q_out, k_out: 0 = F32, 1 = F16, 30 = BF16 */
    int32_t nh;
    int32_t nkv;
    int32_t hd;
    int32_t rot_dim; /* the first rot_dim elements of a head turn, the rest stays (even, 0 .. hd) */
    int32_t layout;  /* B2_ROPE_INTERLEAVED or B2_ROPE_HALF */
    float scale;     /* factor on cos and sin; 0 = 1 */
    int32_t reserved;
    int64_t q_stride;
    int64_t k_stride;
    int64_t v_stride;
    int64_t q_out_stride;
    int64_t k_out_stride;
} b2_rope_rows;

/* transformer.go:936-951 applyRoPE on rows at positions[n_tok]: pair i turns
 * by positions * freqs[i] (freqs [rot_dim / 2] device doubles), the angle
 * reduced in 64 bits, the rotation in fp32, rounded once.  q -> q_out, k ->
 * k_out; either pair may be NULL; a row may be rotated in place (q_out = q
 * with the same stride), other overlaps are not allowed. */
int b2_rope(const b2_rope_rows* rows, const double* freqs, const int32_t* positions, int32_t n_tok, const void* q,
            const void* k, void* q_out, void* k_out, void* stream);
/* The same, with k (rotated) and v written to the cache at slots[n_tok] (page
 * * page_size + place, as b2_page_plan gives them; a slot below 0 or past the
 * cache writes nothing).  q and q_out may be NULL.  The cache's type is the
 * rows', or F16 / BF16 for F32 rows.  No two tokens may share a slot, and no
 * two places of the cache an element: taken from the smallest up, each of the
 * strides, and the distance of k and v, passes the extent of the ones before
 * (B2_ERR_BAD_ARG otherwise; attention only reads, and takes any strides). */
int b2_rope_append(const b2_rope_rows* rows, const b2_paged_kv* kv, const double* freqs, const int32_t* positions,
                   const int64_t* slots, int32_t n_tok, const void* q, const void* k, const void* v, void* q_out,
                   void* stream);

typedef struct {
    int32_t dtype;     /* q and out: 0 = F32, or the cache's type */
    int32_t nh;        /* query heads, a multiple of the cache's nkv */
    int32_t n_req;     /* rows of the table */
    int32_t max_pages; /* entries of a table row */
    int32_t len_add;   /* added to every lens entry */
    int32_t window;    /* > 0: a row sees its last `window` positions only */
    float scale;       /* 0 = 1 / sqrt(hd) */
    float softcap;     /* > 0: s -> softcap * tanh(s / softcap) */
    const float* slopes; /* [nh] device, or NULL: s += slope * (position - last position) */
    int64_t q_stride;     /* elements from row to row; 0 = nh * hd */
    int64_t out_stride;   /* 0 = nh * hd */
    int64_t table_stride; /* 0 = max_pages */
} b2_paged_attn_opts;

/* transformer.go:663-685 attention of `batch` query rows over the paged cache:
 * row b of q ([batch] rows of nh * hd) attends over the first lens[b] +
 * len_add positions of the sequence in table row req[b] (req NULL: b).  With
 * lens = the plan's positions, len_add = 1 and req = its token_req the rows
 * are a step's tokens, prompts included (each row reads its positions for
 * itself, so a long prompt costs its length squared in reads).  The order per
 * score is scale, softcap, slope, mask; fp32 softmax.  Writes out and, when
 * lse is not NULL,
 * lse[b][nh] = log of the sum of e^score.  A row that sees nothing (length <=
 * 0, req < 0) gets zeros and -inf.  A row whose length passes its table or
 * 2^31 - 64, whose req is n_req or more, or whose visible pages are not all in
 * 0 .. n_pages - 1 gets NaN.  Keys and values that are not seen may hold
 * anything; an infinite value that is seen makes its element infinite or NaN.
 * Pages outside the window are not looked at.  d_scratch:
 * b2_attention_paged_scratch_bytes(batch, nh, nkv, hd) bytes of device memory
 * on 16 bytes, no contents needed. */
int64_t b2_attention_paged_scratch_bytes(int32_t batch, int32_t nh, int32_t nkv, int32_t hd);
int b2_attention_paged(const b2_paged_kv* kv, const b2_paged_attn_opts* opts, const void* q, const int32_t* table,
                       const int32_t* lens, const int32_t* req, int32_t batch, void* out, float* lse,
                       void* d_scratch, void* stream);

/* Log probabilities of given tokens, the entropy and the top alternatives of
 * rows of n logits (row i at logits + i * ld, ld >= n; n up to 2^30): the
 * softmax of transformer.go:959-974 kept as logarithms, fp32 sums.
 * logprob[i][m] = log p(ids[i][m]) (an id outside 0 .. n - 1: NaN),
 * entropy[i] in nats (may be NULL), top_ids / top_logprob[i][k] = the k
 * largest logits in order, equal ones by lowest id (k up to 64 and n).  A
 * logit of -inf is a token left out: log p = -inf, nothing added to the
 * entropy.  A row with a NaN or +inf, or with -inf alone, gets NaN for all but
 * top_ids; NaN logits are never alternatives (a place left empty for that
 * gets id -1). */
int b2_logprobs(const void* logits, int32_t dtype, int32_t n, int32_t rows, int64_t ld, const int32_t* ids, int32_t m,
                float* logprob, float* entropy, int32_t k, int32_t* top_ids, float* top_logprob, void* stream);

/* ---- beam search over the paged cache: choose, fork, attend ----
 *
 * A server that keeps several continuations (beams) of each request runs, per
 * step: b2_beam_select picks the best continuations from the step's logits and
 * b2_beam_reorder brings the token histories into their order; b2_page_fork
 * gives every new beam the block table of the beam that it continues, b2_page_copy
 * copies the pages that the two must not share, in all layers at once, and
 * b2_page_pool lists the pages that no row holds any longer; b2_page_plan and
 * b2_rope_append place the new tokens, and b2_page_pool once more (the table
 * and lengths that the plan wrote) takes the plan's pages off the list, which
 * the plan leaves as it was; b2_attention_shared attends, reading what
 * the rows of a request share once.  b2_page_compact, now and then, moves the
 * pages in use to the front of the pool.  Conventions as for the paged serving
 * step above: device pointers on the current device, asynchronous, no
 * allocation, no state between calls, capturable; outputs share no memory with
 * inputs or one another unless said otherwise.  The Go engine runs one
 * sequence with one continuation: no counterpart there. */

/* The k best continuations of each of n_groups requests.  The logits have
 * n_groups * width rows of n (row i at logits + i * ld, ld >= n; dtype 0, 1 or
 * 30), the beams of a request one after another; scores[row] is the sum of a
 * beam's log probabilities so far (NULL: all 0).  The candidate (row, v) has
 *   scores[row] + logits[row][v] - log(sum of e^logits[row]),
 * and parent / token / score [n_groups][k] get the k largest in order, equal
 * ones by lowest row, then lowest v (parent: the row, counted over all
 * requests).  The order is that of sums in 64 bits.  score has fp32
 * exponentials behind it: off by up to 2^-18, as a rule by less than its own
 * rounding, and rounded once.  Candidates of two beams closer than 2^-17 cost their
 * request sums in 64 bits, one beam after another (25 us each for 128256 logits).  Nothing continues with a logit of
 * -inf, from a beam whose score is -inf, +inf or NaN, whose logits hold a NaN
 * or +inf or are all -inf; places that are left get -1, -1, -inf.  eos >= 0
 * (below n): no candidate has that token; its own score in every row, as close,
 * goes to eos_score[rows] (may be NULL; -inf where the row offers none).
 * width, k up to 64, k up to n, n up to 2^30.  d_scratch: b2_beam_select_scratch_bytes(...) bytes on 16
 * bytes, no contents needed. */
int64_t b2_beam_select_scratch_bytes(int32_t n, int32_t n_groups, int32_t width, int32_t k);
int b2_beam_select(const void* logits, int32_t dtype, int32_t n, int32_t n_groups, int32_t width, int64_t ld,
                   const float* scores, int32_t k, int32_t eos, int32_t* parent, int32_t* token, float* score,
                   float* eos_score, void* d_scratch, void* stream);

/* Rows of state in the order of the beams that go on: row r of dst (of n_dst)
 * becomes row parent[r] of src (n_src rows), row_words 32-bit words, rows
 * strides words apart.  lens [n_src] (may be NULL): only the first
 * min(lens[parent[r]], row_words) words are copied, and token [n_dst] (may be
 * NULL) is written behind them where there is room.  new_lens [n_dst] (may be
 * NULL): the words that row r then holds.  A parent outside 0 .. n_src - 1:
 * the row is left as it was, its length 0. */
int b2_beam_reorder(const void* src, int32_t n_src, int64_t src_stride, void* dst, int32_t n_dst, int64_t dst_stride,
                    int64_t row_words, const int32_t* parent, const int32_t* lens, const int32_t* token,
                    int32_t* new_lens, void* stream);

#define B2_FORK_BAD_PARENT 16 /* info[0] of b2_page_fork: a parent of n_src or more */

/* Block tables of rows that continue other rows.  Row s (of n_src, at most
 * 16384) of table holds lens[s] positions in its first ceil(lens[s] /
 * page_size) entries; new row r (of n_req, at most 16384) continues row
 * parent[r] (below 0: it is empty).  Full pages are shared.  A page that is
 * partly filled is written next, so it may have one holder: the first new row
 * of its parent keeps it where refs[page] (NULL: 1 for all) is at most 1,
 * every other gets the next page from the front of free_pages (*n_free of
 * them), in the order of the new rows.  Writes
 *   new_table  [n_req] rows, new_stride apart: the entries in use, nothing else
 *   new_lens   [n_req]
 *   pairs      [n_req][3]: page, copy, positions to copy, one for every page
 *              taken, for b2_page_copy
 *   info       [4] {status, pages taken (pairs), 0, 0}
 * What does not fit (status: B2_PLAN_BAD_LENGTH a negative length,
 * B2_PLAN_TABLE_FULL one past max_pages pages, B2_PLAN_NO_PAGES,
 * B2_FORK_BAD_PARENT) writes nothing but info. */
int b2_page_fork(const int32_t* parent, int32_t n_req, const int32_t* table, int64_t table_stride, const int32_t* lens,
                 int32_t n_src, int32_t page_size, const int32_t* refs, int32_t n_pages, const int32_t* free_pages,
                 const int32_t* n_free, int32_t* new_table, int64_t new_stride, int32_t max_pages, int32_t* new_lens,
                 int32_t* pairs, int32_t* info, void* stream);

/* Copies pages of a cache of `layers` layers (layer l's k and v lie l *
 * layer_stride elements behind kv's, layer_stride a multiple of 8): for each
 * of the first min(*n_pairs, max_pairs) triples of pairs the first pairs[i][2]
 * positions of page pairs[i][0] to page pairs[i][1].  A triple with a page
 * outside the cache, or of one page twice, copies nothing.  No page is written
 * twice, or read and written.  The cache's places must be apart, as for
 * b2_rope_append, and the layers too. */
int b2_page_copy(const b2_paged_kv* kv, int32_t layers, int64_t layer_stride, const int32_t* pairs,
                 const int32_t* n_pairs, int32_t max_pairs, void* stream);

/* Who holds the pool's pages: refs[n_pages] = how many of the n_req rows (at
 * most 16384) hold each page among their first ceil(lens / page_size) entries
 * (at most max_pages; an id outside the pool counts nowhere), free_pages (room for n_pages) = the
 * pages that none holds, ascending, *n_free of them, nothing written past
 * those.  A row is freed by a length of 0; a prefix is kept for later by a row
 * of its own.  d_scratch: b2_page_pool_scratch_bytes(n_pages) bytes on 16
 * bytes. */
int64_t b2_page_pool_scratch_bytes(int32_t n_pages);
int b2_page_pool(const int32_t* table, int64_t table_stride, const int32_t* lens, int32_t n_req, int32_t page_size,
                 int32_t max_pages, int32_t* refs, int32_t n_pages, int32_t* free_pages, int32_t* n_free,
                 void* d_scratch, void* stream);

/* Moves the pages in use to the front of the pool.  With U pages in use (refs
 * > 0, as b2_page_pool leaves them), the i-th highest page of those at U or
 * above goes to the i-th lowest free page below U, for the first min(moves,
 * max_pairs) of them.  The entries in use of the table's rows are changed in
 * place; pairs [max_pairs][3] = page, new page, page_size, for b2_page_copy;
 * info [4] = {0, pairs, U, one past the last page in use afterwards}.  refs
 * stays as it was: b2_page_pool again counts the new pages. */
int64_t b2_page_compact_scratch_bytes(int32_t n_pages);
int b2_page_compact(int32_t* table, int64_t table_stride, const int32_t* lens, int32_t n_req, int32_t page_size,
                    int32_t max_pages, const int32_t* refs, int32_t n_pages, int32_t* pairs, int32_t max_pairs,
                    int32_t* info, void* d_scratch, void* stream);

/* b2_attention_paged for rows that share what they read.  The rows starts[g]
 * .. starts[g + 1] - 1 (starts [n_groups + 1] ascending, on the device) are
 * group g, and the tables of the rows of a group that see anything hold the
 * same pages for the positions below prefix[g] (device): the beams of a
 * request, requests behind one system prompt, or, with b2_page_plan's starts
 * and lens as starts and prefix, the tokens of each request, prompts included.
 * Such positions are read once for all the rows of a group (for every 128 (row, query
 * head) pairs of a KV head), the positions behind them row by row.  Every row
 * sees what it sees in b2_attention_paged, whose other arguments and results
 * these are: lengths, windows, slopes, rows that see nothing (zeros and -inf),
 * rows that get NaN; no row is touched by another's pages, lengths or values.
 * Rows in no group attend alone.  out, lse or d_scratch on one another or on an
 * input is refused (B2_ERR_BAD_ARG).  Groups whose starts do not ascend give rows
 * without meaning, no access out of range.  Scores, softmax and sums are fp32;
 * the products take the probabilities of 16-bit rows in two terms of the
 * cache's type (16 bits of BF16, 22 of F16), of fp32 rows in 22 bits or more.  Every
 * row runs for itself, as in b2_attention_paged, where the head dimension is
 * past 128, where groups have fewer than two rows on average, and where batch *
 * positions * hd * max(nh, 8 * nkv) is at most 2^28 (positions: the window, or max_pages
 * * page_size if that is less), which is faster there; so max_pages should be no
 * more than a step may need.  d_scratch:
 * b2_attention_shared_scratch_bytes(batch, nh, nkv, hd) bytes on 16 bytes, no
 * contents needed. */
int64_t b2_attention_shared_scratch_bytes(int32_t batch, int32_t nh, int32_t nkv, int32_t hd);
int b2_attention_shared(const b2_paged_kv* kv, const b2_paged_attn_opts* opts, const void* q, const int32_t* table,
                        const int32_t* lens, const int32_t* req, int32_t batch, const int32_t* starts,
                        const int32_t* prefix, int32_t n_groups, void* out, float* lse, void* d_scratch, void* stream);

/* ---- tensor parallelism (engine.go LoadOptions.NumGPU; no counterpart in the
 * Go engine, which runs on CPU cores) ----
 *
 * One process per GPU loads the same GGUF with b2_load_opts.tp_size = N and
 * its own tp_rank: it keeps its heads' q / k / v rows and Wo columns, its
 * share of the FFN (gate / up rows, down columns, at 32-block granularity)
 * and of the lm_head vocab rows.  After Wo and after down every rank writes
 * its partial sums into every rank's exchange buffer over NVLink (peer
 * stores) and sums all ranks' partials in rank order, so the residual stream
 * is identical on every rank; the argmax is taken over all ranks' vocab
 * shares the same way.  Before the first forward call, every rank passes the
 * 64-byte handle from b2_tp_handle to the others (any host channel) and calls
 * b2_tp_connect with all N handles in rank order.  Every rank must then make
 * the same sequence of forward calls with the same tokens.  b2_forward's
 * logits_out receives this rank's vocab share (b2_config.vocab_begin /
 * vocab_local); sampling other than greedy is not available. */
int b2_tp_handle(const b2_model* m, void* handle_out);
int b2_tp_connect(b2_model* m, const void* handles);

/* The slices of the GGUF tensors that rank `rank` of a tp-way tensor-
 * parallel model keeps, as b2_load computes them (host arithmetic, no GPU):
 * query heads and KV heads evenly (rows of attn_q / attn_k / attn_v and
 * their biases, input columns of attn_output), the FFN at 32-element block
 * granularity (rows of ffn_gate / ffn_up, input columns of ffn_down; uneven
 * shares allowed), the lm_head by vocab rows.  Fails with B2_ERR_BAD_ARG
 * when the heads do not divide by tp or a share would be empty.  No
 * reference counterpart (the Go engine runs on CPU cores). */
typedef struct {
    int32_t q_row0, q_rows;          /* attn_q rows; attn_output input columns */
    int32_t kv_row0, kv_rows;        /* attn_k / attn_v rows */
    int32_t ffn_row0, ffn_rows;      /* ffn_gate / ffn_up rows; ffn_down input columns */
    int32_t vocab_row0, vocab_rows;  /* lm_head (output or token_embd) rows */
} b2_tp_share;
int b2_tp_share_of(int32_t hidden, int32_t heads, int32_t kv_heads, int32_t ffn, int32_t vocab, int32_t tp,
                   int32_t rank, b2_tp_share* out);

/* Device-side error code of the last launch on this model (B2_ERR_TIMEOUT
 * after a bounded wait gave up), 0 if none; clears it. */
int b2_device_status(b2_model* m);

/* Phase timeline of one decode step (profiling): runs `token` at the current
 * position like b2_forward_argmax and records globaltimer stamps (ns) for
 * every phase, slot and CTA into out_ns[phase][13][cta]: slots 0-3 = consumer
 * wait start, wait done, input staged, work done; 4-5 = producer first and
 * last weight copy issued (0 when the phase has no weights); 6 = total ns the
 * CTA's consumer warps spent waiting for weight chunks, 7 = how many of those
 * waits took longer than 256 ns; 8 = ns the producer waited for free ring
 * slots, 9 = weight chunks it issued; 10 = consumer rows loop done; 11 = total
 * ns the consumer warps spent in tile dot products; 12 = epilogue constants
 * ready.  cap is the
 * capacity of out_ns in elements.  No reference counterpart (the Go engine
 * only logs durations, transformer.go:305-308). */
int b2_trace_step(b2_model* m, int32_t token, int64_t* out_ns, int64_t cap, int32_t* n_phases, int32_t* n_ctas);

/* The cudaStream_t every launch of this model is issued on (for timing with
 * CUDA events on the launching stream).  No reference counterpart. */
void* b2_stream_handle(const b2_model* m);

/* Test hook for failure detection without a GPU fault: the next decode launch
 * waits for `skew` more grid arrivals than will ever come, so its bounded
 * waits run out (about 2 s) and it reports B2_ERR_TIMEOUT through
 * b2_device_status while the context stays usable.  0 disables.  No
 * reference counterpart. */
int b2_debug_wait_skew(b2_model* m, int32_t skew);

/* Test hook for allocation failures: the nth device allocation that
 * b2_load makes from now on (1 = the next one) fails as if cudaMalloc had
 * returned an error, so the caller sees B2_ERR_OOM and can check that the
 * failed load freed everything it had taken.  The hook disarms itself after
 * firing; 0 disarms it.  Process-wide.  No reference counterpart (the Go
 * engine's allocations cannot fail short of a runtime panic). */
int b2_debug_fail_alloc(int32_t nth);

#ifdef __cplusplus
}
#endif
#endif
