/*
 * pbx.h -- C ABI of the MI355X (gfx950) backend for PureBee's quantized
 * matmul / matvec instruction.
 *
 * Every entry point is `extern "C"`, takes plain pointers and sizes, and
 * returns an int status (PBX_OK == 0, negative PBX_E* on failure).  The
 * message for the last failure is returned by pbx_last_error(ctx)
 * (pbx_last_error(NULL) for failures that happen before a context exists).
 * Arguments are validated on the host before any HIP call, so every error
 * path can be exercised without a GPU.
 *
 * Weight orientation is GGUF's: a weight is N rows (output features) of K
 * columns (input features), row n holding K/32 consecutive blocks
 * (gguf.js:36-49; streaming-loader.js:257-259 reads N = dims[1], K = dims[0]).
 *
 * The reference interface each entry point replaces is cited beside it
 * (file:line in sammcj/purebee).  The reference is JavaScript: its "ABI" is
 * the JS module surface of wasm-q4.js, engine.js and purebee.js, which the
 * N-API addon (purebee_amd/napi) and the JS modules (purebee_amd/js) expose
 * on top of this header.
 */
#ifndef PBX_H
#define PBX_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes -------------------------------------------------- */
#define PBX_OK        0
#define PBX_EINVAL   -1   /* bad argument (shape, size, null pointer, type) */
#define PBX_ENODEV   -2   /* no HIP device / device index out of range      */
#define PBX_ENOMEM   -3   /* device or pinned host allocation failed         */
#define PBX_EHIP     -4   /* a HIP runtime call failed                       */
#define PBX_ENOTSUP  -5   /* shape or type not supported by any kernel       */
#define PBX_ELOAD    -6   /* code object missing or not loadable (hipModuleLoad) */
#define PBX_EIO      -7   /* a file could not be opened or mapped            */
#define PBX_ETIMEOUT -8   /* a bounded device-side wait gave up: data that one
                             workgroup publishes for another inside a launch
                             never arrived; the call's results are invalid   */

/* ---- weight types ----------------------------------------------------
 * GGML numbering, as gguf.js:30-33 (GGML_TYPE).  PBX_TYPE_Q8_REF is the
 * reference's own in-memory Q8 tensor (quantize.js:30-50, QuantizedTensor
 * 'q8_0'): int8 values of a [K,N] matrix laid out flat, one f32 scale per
 * 32 consecutive flat elements, consumed by matmul_q8 (quantize.js:224-266).
 */
#define PBX_TYPE_F32     0
#define PBX_TYPE_F16     1
#define PBX_TYPE_Q4_0    2
#define PBX_TYPE_Q4_1    3
#define PBX_TYPE_Q8_0    8
#define PBX_TYPE_Q6_K    14
#define PBX_TYPE_Q8_REF  100

typedef struct pbx_ctx pbx_ctx;
typedef struct pbx_weight pbx_weight;

/* ---- context ----------------------------------------------------------
 * Replaces wasmQ4.init() (wasm-q4.js:647-668) / engine.initWasm()
 * (engine.js:28-31): selects the device, creates the context's stream and
 * loads the gfx950 code object with hipModuleLoad.  A context is used from
 * one host thread at a time (the reference calls everything from the main
 * JS thread, thread-pool.js:3-7).
 */
int         pbx_init(int device, pbx_ctx **out);
void        pbx_shutdown(pbx_ctx *ctx);
const char *pbx_last_error(const pbx_ctx *ctx);
/* Device name (NUL-terminated, truncated to cap) and compute-unit count. */
int         pbx_device_info(pbx_ctx *ctx, char *name, size_t cap, int *cu_count);

/* ---- resident weights ------------------------------------------------
 * Replaces the per-call copy of the raw block bytes into WASM memory
 * (wasm-q4.js:735-738) and wasmSimd.allocWeights / engine.cacheWeight
 * (wasm-simd.js:406-414, engine.js:39-42): the bytes are copied to the GPU
 * once through pinned staging buffers and repacked there into the layout
 * the kernels read; the handle stays valid until pbx_weight_free.
 *
 * host/nbytes hold GGUF row-major blocks: N rows of K/32 blocks of
 * 18 B (Q4_0: fp16 d + 16 nibble bytes), 20 B (Q4_1: fp16 d, fp16 m +
 * 16 nibble bytes) or 34 B (Q8_0: fp16 d + 32 int8), or of K/256 blocks of
 * 210 B (Q6_K: ql[128], qh[64], int8 scales[16], fp16 d), gguf.js:36-49 and
 * 239-364; for PBX_TYPE_F32 / PBX_TYPE_F16, N*K little-endian floats /
 * halves.  K must be a multiple of 32 for every type (256 for Q6_K).
 */
int pbx_weight_upload(pbx_ctx *ctx, int type, int64_t N, int64_t K,
                      const void *host, size_t nbytes, pbx_weight **out);
/* The reference's QuantizedTensor 'q8_0' of shape [K,N] (quantize.js:30-50):
 * q = K*N int8 values, scales = ceil(K*N/32) f32 values. */
int pbx_weight_upload_q8ref(pbx_ctx *ctx, int64_t K, int64_t N,
                            const int8_t *q, const float *scales,
                            int64_t n_scales, pbx_weight **out);
/* Replaces wasmSimd.resetWeights (wasm-simd.js:511-513) / PureBee.FREE
 * (purebee.js:200-202) for a resident weight. */
int pbx_weight_free(pbx_ctx *ctx, pbx_weight *w);
int pbx_weight_info(const pbx_weight *w, int *type, int64_t *N, int64_t *K,
                    size_t *device_bytes);

/* ---- the instruction -------------------------------------------------
 * Y[M,N] = X[M,K] . W^T (+ bias[N]), fp32 in and out.
 *   M == 1   -> fused unpack/dequant/dot GEMV (one wavefront per row group)
 *   M >= 2   -> dequant -> LDS -> fp16 MFMA GEMM (quantized types)
 * Replaces, with the same arithmetic meaning:
 *   wasmQ4.q4_0_matvec(x, rawBuf, N, K)           wasm-q4.js:716-747
 *   quantizedMatvec(x, rawBuf, type, N, K)        llama-streaming.js:168-177
 *   AtomicsThreadPool.matvec(...)                 thread-pool.js:165-246
 *   wasmQ4.lmHead(hidden, emb, vocab, dim) (F32)  wasm-q4.js:798-839
 *   engine.tensorMulAdd(x, W, b)  (F32)           engine.js:180-244
 *   engine.tensorMulAddQ8(x, Wq, b) (Q8_REF)      engine.js:259-269,
 *                                                 quantize.js:224-266
 * pbx_linear takes host pointers and blocks until Y is written (the
 * reference's synchronous convention, wasm-q4.js:744-746).  pbx_linear_dev
 * takes device pointers and only enqueues on the context's stream.
 * bias may be NULL.
 */
int pbx_linear(pbx_ctx *ctx, const pbx_weight *W, const float *X, int64_t M,
               const float *bias, float *Y);
int pbx_linear_dev(pbx_ctx *ctx, const pbx_weight *W, const float *dX,
                   int64_t M, const float *dBias, float *dY);
/* pbx_linear_dev that allocates nothing: no counterpart in the reference.
 * For callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  The same
 * kernels and results as pbx_linear_dev; the M >= 4 GEMM's activation pair,
 * row scales and split-K partials live in one static device array of
 * PBX_NOALLOC_WORKSPACE_BYTES per GPU (held until the process ends) instead
 * of the context's grow-only buffers.  A shape that needs more workspace
 * fails with PBX_EINVAL.  Calls on one GPU share that array: calls that
 * overlap on one GPU (other contexts or streams) race. */
#define PBX_NOALLOC_WORKSPACE_BYTES (64u << 20)
int pbx_linear_dev_noalloc(pbx_ctx *ctx, const pbx_weight *W, const float *dX, int64_t M,
                           const float *dBias, float *dY);
/* Introspection for the two above, no reference counterpart (tests and
 * capacity planning): *grown_bytes = device workspace the allocating entry
 * points of this context have allocated so far (the noalloc one never adds
 * to it), *static_bytes = the static workspace of the noalloc one (0 when
 * it is unavailable); pbx_ctx_stream = the context's HIP stream (a
 * hipStream_t), on which every enqueueing entry point works, for callers
 * that capture that work into a graph or order their own work after it. */
int   pbx_workspace_info(const pbx_ctx *ctx, size_t *grown_bytes, size_t *static_bytes);
void *pbx_ctx_stream(const pbx_ctx *ctx);

/* Exact dequantisation of a resident weight to fp32, row-major [N,K]
 * (for PBX_TYPE_Q8_REF: [K,N], the reference's own orientation).
 * Replaces loadTensorData's Q4_0/Q8_0 branches (gguf.js:239-286) and
 * dequantize_q8 (quantize.js:170-181).  Bit-exact by construction. */
int pbx_dequant(pbx_ctx *ctx, const pbx_weight *W, float *Y);
int pbx_dequant_dev(pbx_ctx *ctx, const pbx_weight *W, float *dY);

/* ---- host-side quantisers (CPU) ---------------------------------------
 * Q8_0 with the numerics of quantize_q8 (quantize.js:79-109: absmax/127,
 * ECMAScript Math.round of x*127/absmax in double) applied per 32-block
 * along K of each row, the scale stored as fp16 (GGUF Q8_0 layout).
 * Q4_0 with d = absmax/8 stored as fp16 and nibble = clamp(round(x*8/absmax),
 * -8, 7) + 8, GGUF non-interleaved nibble order (gguf.js:259-286).
 * Q4_1 with d = (max-min)/15 and m = min stored as fp16 and nibble =
 * clamp(round((x-m)/d), 0, 15) against the stored values (GGUF Q4_1 layout,
 * gguf.js:288-314).  The reference reads Q4_1 but has no quantiser for it.
 * Q6_K (gguf.js:317-364 layout) with sub-block scales absmax/31 rounded
 * to int8 steps of d = max/127 (fp16) and codes clamp(round(x/(d*sc)),
 * -32, 31) + 32; the reference reads Q6_K but has no quantiser for it.
 * out must hold N*K/32*34 (Q8_0), N*K/32*18 (Q4_0), N*K/32*20 (Q4_1) or
 * N*K/256*210 (Q6_K, K % 256 == 0) bytes. */
int pbx_quantize_q8_0(const float *w, int64_t N, int64_t K, uint8_t *out);
int pbx_quantize_q4_0(const float *w, int64_t N, int64_t K, uint8_t *out);
int pbx_quantize_q4_1(const float *w, int64_t N, int64_t K, uint8_t *out);
int pbx_quantize_q6_k(const float *w, int64_t N, int64_t K, uint8_t *out);
/* quantize_q8 itself (quantize.js:79-109): flat, f32 scales (Q8_REF). */
int pbx_quantize_q8_ref(const float *w, int64_t n, int8_t *q, float *scales);

/* Seeded synthetic data: element i of the stream is a pure function of
 * (seed, i): SplitMix64 -> Box-Muller in double -> mean + std*z as float. */
int pbx_synth_normal(uint64_t seed, int64_t n, double mean, double std,
                     float *out);

/* ---- device memory, streams, timing (for callers on device pointers) -- */
int pbx_dev_alloc(pbx_ctx *ctx, size_t bytes, void **out);
int pbx_dev_free(pbx_ctx *ctx, void *p);
int pbx_memcpy_h2d(pbx_ctx *ctx, void *dst, const void *src, size_t bytes);
int pbx_memcpy_d2h(pbx_ctx *ctx, void *dst, const void *src, size_t bytes);
int pbx_memset_dev(pbx_ctx *ctx, void *dst, int value, size_t bytes);
/* Device-to-device copy by a plain kernel (bytes and both addresses 16-byte
 * aligned): a known-traffic kernel for calibrating hardware byte counters.
 * No reference counterpart. */
int pbx_dev_copy(pbx_ctx *ctx, void *dst, const void *src, size_t bytes);
int pbx_sync(pbx_ctx *ctx);
/* HIP events recorded on the context's stream: the kernels' own stream. */
int pbx_timer_start(pbx_ctx *ctx);
int pbx_timer_stop(pbx_ctx *ctx, double *elapsed_ms);
/* Enqueue `reps` passes over n_ops (W[i], dX[i] -> dY[i]) linears at row
 * count M and return the elapsed time between HIP events recorded on the
 * context's stream around the whole sequence. */
int pbx_bench_linear(pbx_ctx *ctx, int n_ops, const pbx_weight *const *W,
                     const float *const *dX, float *const *dY, int64_t M,
                     int reps, double *elapsed_ms);
/* The same pass captured once into a HIP graph and replayed `reps` times
 * (the launches stream without host launch gaps).  Timing helpers; no
 * reference counterpart. */
int pbx_bench_linear_graph(pbx_ctx *ctx, int n_ops, const pbx_weight *const *W,
                           const float *const *dX, float *const *dY, int64_t M,
                           int reps, double *elapsed_ms);

/* ---- resident model and on-GPU decode step ----------------------------
 * A Llama-family model held in device memory, replacing the reference's
 * runtimes for decode: LlamaRuntime.forward (llama.js:204-371) and
 * StreamingLlamaRuntime.forward/_runLayerQ4 (llama-streaming.js:505-606,
 * 738-815): RMSNorm (eps), q/k/v, RoPE on adjacent pairs with theta,
 * KV cache, grouped-query attention, output projection + residual, RMSNorm,
 * SwiGLU FFN + residual; final RMSNorm, LM head, greedy argmax (first
 * maximum, llama.js:432-442).  Activations and the KV cache are fp32.
 */
typedef struct pbx_model pbx_model;

typedef struct pbx_model_config {
  int32_t dim, hidden_dim, n_layers, n_heads, n_kv_heads, head_dim;
  int32_t vocab_size, max_seq;
  int32_t weight_type;  /* every layer matrix: any PBX_TYPE_* but Q8_REF    */
  int32_t embed_type;   /* token_embd (row lookup and, when tied, LM head) */
  int32_t output_type;  /* untied LM head type, or -1: tied to token_embd  */
  float rms_eps;        /* 1e-5 in the reference (purebee.js:164)         */
  double rope_theta;    /* 10000 (llama.js:33) or the GGUF rope.freq_base */
} pbx_model_config;

/* Tensor ids for pbx_model_set_tensor, named as the GGUF tensors they take
 * (gguf.js:378-410).  Matrices are GGUF row-major blocks of their type,
 * [N rows = out features][K = in features]; norms are f32. */
#define PBX_T_TOKEN_EMBD   0   /* [vocab, dim]   embed_type            */
#define PBX_T_OUTPUT       1   /* [vocab, dim]   output_type (untied)  */
#define PBX_T_OUTPUT_NORM  2   /* [dim] f32                            */
#define PBX_T_ATTN_NORM    3   /* per layer: [dim] f32                 */
#define PBX_T_FFN_NORM     4   /* per layer: [dim] f32                 */
#define PBX_T_ATTN_Q       5   /* per layer: [dim, dim]                */
#define PBX_T_ATTN_K       6   /* per layer: [kv_dim, dim]             */
#define PBX_T_ATTN_V       7   /* per layer: [kv_dim, dim]             */
#define PBX_T_ATTN_OUTPUT  8   /* per layer: [dim, dim]                */
#define PBX_T_FFN_GATE     9   /* per layer: [hidden, dim]   (w1)      */
#define PBX_T_FFN_UP      10   /* per layer: [hidden, dim]   (w3)      */
#define PBX_T_FFN_DOWN    11   /* per layer: [dim, hidden]   (w2)      */

int pbx_model_create(pbx_ctx *ctx, const pbx_model_config *cfg, pbx_model **out);
int pbx_model_free(pbx_model *m);
/* Replaces the loaders' per-tensor reads (streaming-loader.js:245-299,
 * loadResidentWeights 324-335): one upload, resident afterwards. */
int pbx_model_set_tensor(pbx_model *m, int tensor, int layer, const void *data,
                         size_t nbytes);
/* forward(tokenIds, startPos) (llama.js:204, llama-streaming.js:738):
 * runs tokens[0..n) at positions start_pos.., writing the KV cache; returns
 * the last position's logits (if logits != NULL, [vocab]) and its argmax. */
int pbx_model_forward(pbx_model *m, const int32_t *tokens, int n_tokens,
                      int start_pos, float *logits, int32_t *next_token);
/* StreamingLlamaRuntime.forward(tokenIds, startPos, {maxLayers})
 * (llama-streaming.js:738-815): as pbx_model_forward, but only the first
 * max_layers layers run (0: all of them, `maxLayers || nLayers`; the limit
 * is min(max_layers, n_layers)), then the final RMSNorm and the LM head on
 * their output; the KV cache of the later layers is not written at these
 * positions.  *layers_used (if not NULL) receives the layers run, the
 * `layersUsed` of the reference's result. */
int pbx_model_forward_layers(pbx_model *m, const int32_t *tokens, int n_tokens,
                             int start_pos, int max_layers, float *logits,
                             int32_t *next_token, int *layers_used);
/* forward() over n tokens in ONE batched pass that keeps every position's
 * output (the reference computes them inside forward, llama.js:204-371, and
 * keeps only the last): logits [n][vocab] (or NULL) and next_tokens[n], the
 * argmax of each row (or NULL).  Quantized matrices run on the MFMA GEMM
 * with all n rows; this is the speculative verify of speculative.js:131-185
 * done as one forward instead of one forward per draft token. */
int pbx_model_forward_batch(pbx_model *m, const int32_t *tokens, int n_tokens,
                            int start_pos, float *logits, int32_t *next_tokens);
/* The greedy decode loop of generate() (llama.js:475-489): feeds `token` at
 * start_pos, then each step's argmax, n_steps times, entirely on the GPU;
 * out_tokens[i] is the token chosen by step i. */
int pbx_model_generate(pbx_model *m, int32_t token, int start_pos, int n_steps,
                       int32_t *out_tokens, float *last_logits);
/* The same loop stopping at the first token in eos_ids[0..n_eos), as
 * llama.js:475-489 stops at eosId (`if (nextToken === eosId) break`):
 * out_tokens receives the *n_out <= max_steps chosen tokens, the EOS last if
 * one was chosen, and the cache holds no row past the position that fed it.
 * Steps run in chunks of whole graph launches, the chunk's tokens checked
 * on the host after each. */
int pbx_model_generate_eos(pbx_model *m, int32_t token, int start_pos, int max_steps,
                           const int32_t *eos_ids, int n_eos, int32_t *out_tokens,
                           int *n_out);
/* resetCache / rollbackCache (llama-streaming.js:828-862): zero cache
 * positions >= pos of every layer. */
int pbx_model_reset_cache(pbx_model *m);
int pbx_model_rollback(pbx_model *m, int pos);
int pbx_model_info(const pbx_model *m, size_t *device_bytes, int *uses_graph);
/* Measurement: n_steps greedy decode steps launched kernel by kernel (no
 * graph), each kernel carrying a start and a stop HIP event that its own
 * dispatch stamps (hipExtModuleLaunchKernel).  op_us[i] is the mean
 * execution time of kernel i (the duration a kernel trace reports, without
 * the gaps between kernels), op_bytes[i] its mean algorithmic bytes (may be
 * NULL); *n_ops is the kernel count per step (arrays hold min(cap, *n_ops)
 * entries).
 * pbx_model_op_name gives "role:kernel" of kernel i (no reference
 * counterpart: the reference has no GPU kernels to profile). */
int pbx_model_profile(pbx_model *m, int32_t token, int start_pos, int n_steps,
                      double *op_us, double *op_bytes, int cap, int *n_ops);
int pbx_model_op_name(const pbx_model *m, int i, char *buf, size_t cap);
/* Test hook, no reference counterpart: makes the attention workgroups of
 * layer `layer`'s joined q|k|v + attention launch wait for cells tagged
 * `skew` epochs ahead (none ever are), giving up after `spin` polls (0: the
 * kernel's default), so that the bounded wait's error path can be tested
 * with every kernel still exiting normally; the call then fails with
 * PBX_ETIMEOUT.  layer < 0 restores the normal launch.  Returns
 * PBX_ENOTSUP when the model's step has no such launch. */
int pbx_model_test_handoff(pbx_model *m, int layer, int skew, int spin);
/* Test hook, no reference counterpart: in the joined launches that split a
 * long context over workgroups, every workgroup expects its peers' states
 * under tags `skew` epochs ahead (none ever arrive) and polls for them
 * `spin` times (0: the kernel's default) before it computes them itself.
 * Results stay the same, bit for bit.  skew 0 restores the normal launch.
 * Returns PBX_ENOTSUP when the model's step has no such launch. */
int pbx_model_test_peers(pbx_model *m, int skew, int spin);
/* Measurement: the GEMV kernels of one role ("qkv", "o", "gate_up", "down",
 * "lm_head") launched back to back over every layer's weights, `reps`
 * passes between two HIP events on the model's stream; returns the mean
 * time and algorithmic bytes per launch.  Leaves the activations in an
 * unspecified state (the next forward re-embeds its token). */
int pbx_model_bench_role(pbx_model *m, const char *role, int reps,
                         double *us_per_launch, double *bytes_per_launch,
                         int *launches_per_rep);

/* ---- GGUF files ----------------------------------------------------------
 * The build's own GGUF v2/v3 reader, replacing GGUFParser and parseHeader
 * (gguf.js:76-194, streaming-loader.js:35-87): the file is mapped read-only,
 * header, metadata and tensor table are parsed with bounds checks, and
 * tensor data is served from the mapping (no copy).  Errors follow the
 * reference's: bad magic, a version outside 2..3, a tensor type the
 * reference cannot size (gguf.js:36-49, 206-213) fail the open.  pbx_gguf_*
 * calls take no context; pbx_last_error(NULL) names the failure.
 */
typedef struct pbx_gguf pbx_gguf;

typedef struct pbx_gguf_tensor {
  const char *name;      /* NUL-terminated, valid until pbx_gguf_close      */
  int32_t type;          /* GGML type id (gguf.js:30-33)                   */
  int32_t n_dims;        /* 1..4                                            */
  int64_t dims[4];       /* GGUF order: dims[0] = row length (K), dims[1] =
                            rows (N); unused dims are 1                     */
  uint64_t offset;       /* absolute file offset of the data                */
  uint64_t nbytes;       /* tensorByteSize (gguf.js:206-213)                */
  const void *data;      /* the bytes, inside the read-only mapping         */
} pbx_gguf_tensor;

int     pbx_gguf_open(const char *path, pbx_gguf **out);
void    pbx_gguf_close(pbx_gguf *g);
int     pbx_gguf_info(const pbx_gguf *g, uint32_t *version, int64_t *n_tensors,
                      int64_t *n_kv, uint64_t *data_start);
int     pbx_gguf_tensor_info(const pbx_gguf *g, int64_t i, pbx_gguf_tensor *out);
int64_t pbx_gguf_find_tensor(const pbx_gguf *g, const char *name);  /* -1: absent */
/* Metadata by key: integers (any integer type or bool), floats (f32/f64 or
 * an integer), strings (pointer into the mapping, not NUL-terminated),
 * arrays (element type and count). */
int pbx_gguf_get_int(const pbx_gguf *g, const char *key, int64_t *out);
int pbx_gguf_get_float(const pbx_gguf *g, const char *key, double *out);
int pbx_gguf_get_string(const pbx_gguf *g, const char *key, const char **str, uint64_t *len);
int pbx_gguf_get_array(const pbx_gguf *g, const char *key, uint32_t *elem_type,
                       uint64_t *count);
/* extractConfig (gguf.js:429-450) under general.architecture with the
 * reference's defaults (head_count_kv = head_count, rms eps 1e-5, rope
 * freq_base 10000); vocab_size = the tokenizer's token count
 * (streaming-loader.js:57) or token_embd's rows; weight/embed/output types
 * from blk.0.attn_q / token_embd / output (-1: tied).  max_seq <= 0 takes
 * min(context_length, 8192). */
int pbx_gguf_model_config(const pbx_gguf *g, int max_seq, pbx_model_config *cfg);
/* loadGGUFModel (gguf.js:778-839) / StreamingLlamaRuntime's loader
 * (streaming-loader.js:245-335) as one step: open, configure, create the
 * model and upload every tensor once, names mapped as gguf.js:378-410.
 * Token embedding and output rows past the vocabulary are not uploaded.
 * Tensors outside the Llama layout, layer matrices of mixed types and
 * shapes that disagree with the metadata are errors. */
int pbx_model_load_gguf(pbx_ctx *ctx, const char *path, int max_seq, pbx_model **out);

/* ---- speculative decoding ----------------------------------------------
 * SelfSpeculativeDecoder.generate (speculative.js:58-204) in its greedy
 * mode, with the draft taken from a separate (smaller) model instead of the
 * target's first layers.  Both caches are reset, the prompt is prefilled
 * into both, then each round drafts up to draft_count tokens with `draft`,
 * verifies them with `target`, accepts the longest agreeing prefix, emits
 * the target's own token at the first disagreement (or a bonus token when
 * every draft agrees) and rolls the target's cache back past the rejected
 * positions.  batched_verify = 1 verifies a round's drafts in one
 * pbx_model_forward_batch (M = drafts + 1); 0 verifies them one forward at
 * a time as the reference does.  Token ids outside a model's vocabulary are
 * taken modulo it (draft and target vocabularies may differ).
 * out_tokens receives the generated tokens (not the prompt): at most
 * max_tokens + 1 of them (the reference's bound), *n_out of them. */
typedef struct pbx_spec_stats {
  int32_t rounds, drafted, accepted;
  double prefill_ms, decode_ms;  /* host wall clock around the two phases */
} pbx_spec_stats;

int pbx_speculative_generate(pbx_model *target, pbx_model *draft, const int32_t *prompt,
                             int n_prompt, int max_tokens, int draft_count,
                             const int32_t *eos_ids, int n_eos, int batched_verify,
                             int32_t *out_tokens, int *n_out, pbx_spec_stats *stats);

/* SelfSpeculativeDecoder.generate (speculative.js:58-204) as the reference
 * runs it, greedy: the draft is the model's own first draft_layers layers
 * (forward([t], pos, {maxLayers: draftLayers}) and argmax, draft_count
 * times, speculative.js:96-111), on its own KV cache; the rest as
 * pbx_speculative_generate with target = draft = m.  Prompt tokens must lie
 * in the vocabulary. */
int pbx_self_speculative_generate(pbx_model *m, const int32_t *prompt, int n_prompt,
                                  int max_tokens, int draft_layers, int draft_count,
                                  const int32_t *eos_ids, int n_eos, int batched_verify,
                                  int32_t *out_tokens, int *n_out, pbx_spec_stats *stats);

/* ---- paged 8-bit KV cache ------------------------------------------------
 * A KV cache that many sequences share, for callers that run several requests
 * through one resident model (no reference counterpart: the reference holds
 * one sequence in f32).  The pool has n_pages pages of page_tokens positions
 * (of every layer); a sequence holds whole pages, handed out by the library as
 * it grows.  Keys and values are int8 codes with one f32 scale s for each
 * block of PBX_KV_BLOCK positions of a sequence, each KV head, keys and values
 * apart:
 *   s = max |x| / 127 over the block's rows, rounded to f32,
 *   code = x / s rounded half to even, and the value it stands for is code * s.
 * Rows appended to a block that already holds some raise s where their own
 * maximum asks for it (it never falls); the earlier codes c are then rounded
 * again, c * s_old / s_new.  Quotients and rotated values are taken in 64 bits,
 * so codes do not depend on the batch that appends a row, only on which rows
 * of a block arrive together.  A scale below 2^-120 is held as 0 (the block
 * reads as zeros); a block that got a NaN or an infinite value reads as NaN.
 */
typedef struct pbx_kv pbx_kv;
typedef struct pbx_kv_batch pbx_kv_batch;

#define PBX_KV_BLOCK 32  /* positions that share a scale */

/* Position rotation of queries and keys: none, of adjacent dims (2i, 2i + 1)
 * as pbx_model rotates (llama.js:159-191), or of dims (i, i + rope_dim / 2).
 * Pair i turns by the angle pos / rope_scale * rope_theta^(-2i / rope_dim) /
 * rope_factors[i], evaluated in 64 bits; dims from rope_dim on are copied. */
#define PBX_ROPE_NONE   0
#define PBX_ROPE_PAIRS  1
#define PBX_ROPE_HALVES 2

typedef struct pbx_kv_config {
  int32_t n_layers, n_heads, n_kv_heads; /* n_kv_heads divides n_heads          */
  int32_t head_dim;      /* 32..256, a multiple of 4                            */
  int32_t page_tokens;   /* 32, 64, 128, 256, 512 or 1024                       */
  int32_t n_pages;
  int32_t max_seqs;      /* sequence ids are 0..max_seqs - 1                    */
  int32_t max_seq;       /* positions of one sequence, at most 2^20             */
  int32_t rope_style;    /* PBX_ROPE_*                                          */
  int32_t rope_dim;      /* leading dims that turn: a multiple of 4, 0: head_dim */
  double rope_theta;     /* > 0                                                 */
  double rope_scale;     /* > 0: positions are divided by it (1: as they are)   */
  const float *rope_factors; /* [rope_dim / 2] or NULL (all 1); > 0; copied     */
} pbx_kv_config;

int pbx_kv_create(pbx_ctx *ctx, const pbx_kv_config *cfg, pbx_kv **out);
/* Frees the cache and every batch of it. */
int pbx_kv_free(pbx_kv *kv);
int pbx_kv_info(const pbx_kv *kv, int *free_pages, size_t *device_bytes);
/* Positions that a sequence holds; and dropping those from n_tokens on (0: the
 * whole sequence), which gives back the pages they leave empty.  Batches that
 * were set over dropped positions are refused from then on. */
int pbx_kv_length(const pbx_kv *kv, int seq, int *n_tokens);
int pbx_kv_truncate(pbx_kv *kv, int seq, int n_tokens);

/* Branches: sequence dsts[i] (none twice) comes to hold the first lens[i] positions
 * (lens == NULL: all) that srcs[i] held before the call, for all i at once, so beams
 * may take each other's places; what dsts[i] held is let go of, as by truncation, and
 * dsts[i] == srcs[i] only shortens.  Nothing is copied: the sequences share pages, which
 * free_pages counts once.  A batch that lengthens a sequence inside a shared page gives
 * it a copy of the page first (pbx_kv_batch_set, from the pool; the last one to hold a
 * page keeps it), and other batches over that sequence have to be set again.  Rows in
 * pages that have come to be shared since their batch was set cannot be appended
 * (PBX_EINVAL), nor can pages be shared to which a captured batch appends.  Waits for
 * no GPU work. */
int pbx_kv_fork(pbx_kv *kv, int n, const int32_t *dsts, const int32_t *srcs, const int32_t *lens);
/* Sequence seqs[i] (none twice) keeps counts[i] of its positions and drops the others;
 * `positions` lists them, rising, one sequence after the other.  The k-th that is kept
 * becomes position k: its key is turned from its old to its new position (with no
 * rotation it stays) and its block is coded anew, as if rows of the values that the old
 * codes stand for were appended together.  Blocks whose rows all stay where they are
 * stay as they are.  A block that gets a row from a block that reads as NaN reads as NaN.
 * Pages from the first row that moves on are written into free pages of the pool, at
 * least one (PBX_ENOMEM, and nothing changed; the fewer there are, the more launches),
 * and given back; sequences that share them keep theirs.  Batches over moved positions
 * are refused from then on.  Enqueues on the context's stream, and waits for no GPU work
 * but the lists of the compaction before.  Where a launch fails (PBX_EHIP) nothing changed,
 * or, if ones before it wrote pages that were given back, the sequences are left with the
 * positions in pages before the first row that moves. */
int pbx_kv_compact(pbx_kv *kv, int n, const int32_t *seqs, const int32_t *counts, const int32_t *positions);

/* A batch: counts[i] rows of sequence seqs[i] (none twice) at the positions
 * starts[i].., packed in this order (all rows of a sequence side by side).
 * pbx_kv_batch_set lengthens a sequence to hold its rows, with pages from the
 * pool (PBX_ENOMEM, and nothing changed, when it has too few); starts[i] is at
 * most its length, and starts == NULL means each sequence's end.  counts[i] may
 * be 0.  The set-up is made once and used by every layer's calls below; it waits
 * for no GPU work but the previous set-up of the same batch (and the context's
 * stream, where a batch larger than any before needs more memory).  The three
 * calls enqueue on the context's stream; of one batch they use the same workspace,
 * so its calls and replays of graphs that captured them run on one stream at a time.
 * A batch whose calls were captured keeps its rows (set refuses, PBX_EINVAL):
 * a replay runs over the same positions, which the sequences must still hold
 * (and, if it appends, end with), and the batch lives as long as the graph (a
 * batch whose capture was thrown away is freed, and another one set).  A call
 * that is refused, or has no rows, holds nothing.
 * Inside a capture no cache or batch is made, set or freed, and no sequence forked or
 * compacted (PBX_EINVAL).
 * Positions that a batch took hold nothing defined until they are appended.
 */
int pbx_kv_batch_create(pbx_kv *kv, pbx_kv_batch **out);
int pbx_kv_batch_free(pbx_kv_batch *b);
int pbx_kv_batch_set(pbx_kv_batch *b, int n_seqs, const int32_t *seqs,
                     const int32_t *starts, const int32_t *counts);
int pbx_kv_batch_rows(const pbx_kv_batch *b, int *n_rows);

/* Rotates the batch's queries and keys by their positions and appends its keys
 * and values to layer `layer`.  Rows are f32 [n_heads | n_kv_heads][head_dim],
 * *_stride floats apart (a multiple of 4; 0: packed); addresses are 16-byte
 * aligned.  The rotated queries go to dQout, which may be dQ itself (dQ and
 * dQout both NULL: keys and values only).  The rows must be the last of their
 * sequences. */
int pbx_kv_append_dev(pbx_kv_batch *b, int layer, const float *dQ, int64_t q_stride,
                      const float *dK, int64_t k_stride, const float *dV, int64_t v_stride,
                      float *dQout, int64_t qout_stride);
/* Attention of the batch's (rotated) query rows over layer `layer` of their
 * sequences: head h of a row at position p sees KV head h / (n_heads /
 * n_kv_heads) at positions 0..p.  scale: of the products (0: 1 /
 * sqrt(head_dim)).  Rows as above; dOut [n_rows][n_heads][head_dim], which may
 * be dQ itself.  Values are used as they stand in the cache and sums are held in
 * f32.  Queries enter with 22 bits (2^-25 of their row's largest at least), a
 * probability with 22 bits, or 2^-30 of the largest in its block of
 * PBX_KV_BLOCK positions where that is more.  Scores (scale q . K) are to stay
 * below 10^8.  The result of a row does not depend on the other rows' values. */
int pbx_kv_attention_dev(pbx_kv_batch *b, int layer, const float *dQ, int64_t q_stride,
                         float scale, float *dOut, int64_t out_stride);
/* The batch's rows of the cache as the values they stand for, f32 [n_rows]
 * [n_kv_heads][head_dim] (either may be NULL). */
int pbx_kv_read_dev(pbx_kv_batch *b, int layer, float *dK, int64_t k_stride, float *dV,
                    int64_t v_stride);

/* ---- log probabilities -----------------------------------------------------
 * Of `rows` rows of f32 logits [vocab], `stride` floats apart (0: vocab):
 *   dLogp[r]     log softmax at dTargets[r] (NaN for a target outside the
 *                vocabulary); NULL, like dTargets, to leave it out
 *   dEntropy[r]  -sum p log p, in nats; or NULL
 *   dTopIds, dTopLogp [rows][top]: the `top` (0..PBX_LOGPROBS_TOP_MAX, at most
 *                vocab) most likely tokens in order, equal logits by the lower
 *                index, and their log probabilities; either NULL to leave it out
 * A logit of -inf is a token that cannot be chosen (log probability -inf, no
 * entropy).  A row with a NaN or +inf logit, or with nothing but -inf, has no
 * distribution: NaN log probabilities and entropy, top tokens -1.
 * Only enqueues on the context's stream.  work: device memory of the size that
 * pbx_logprobs_workspace gives (it may be 0), 16-byte aligned, any content,
 * for this call alone until it has run.  No reference counterpart: the
 * reference samples on the host (llama.js:394-442). */
#define PBX_LOGPROBS_TOP_MAX 32
int pbx_logprobs_workspace(pbx_ctx *ctx, int64_t rows, int64_t vocab, int top, size_t *bytes);
int pbx_logprobs_dev(pbx_ctx *ctx, const float *dLogits, int64_t stride, int64_t rows,
                     int64_t vocab, const int32_t *dTargets, int top, float *dLogp,
                     float *dEntropy, int32_t *dTopIds, float *dTopLogp, void *work,
                     size_t work_bytes);

/* The same of rows whose logits are X . W^T, without keeping those: a piece of the
 * vocabulary at a time.  W: a head of any type but Q8_REF, [vocab, K]; dX [rows][K], at
 * most 65,535 rows, 16-byte aligned.
 *   dLogp[r]     log softmax at dTargets[r] (NaN for a target outside the vocabulary);
 *                NULL, like dTargets, to leave it out
 *   dEntropy[r]  -sum p log p, in nats; or NULL
 *   dLse[r]      log of the sum of all e^logit, which the gradient needs; or NULL
 * A row without a distribution (see above) answers with NaN; weights are finite.
 * Activations enter the logits with 22 bits each (2^-39 of their row's largest at least)
 * or with 22 bits of the largest of 32 columns, as in pbx_linear, or as they are; the
 * weights of an F32 head with 22 bits each (2^-39 of their row's largest at least); sums
 * are held in f32.  Only enqueues on the context's stream.  work: device memory of the size that
 * pbx_linear_logprobs_workspace gives (grad 1: for the gradient), 256-byte aligned, any
 * content, for this call alone until it has run (graphs that may run side by side need
 * one each).  No reference counterpart. */
int pbx_linear_logprobs_workspace(pbx_ctx *ctx, const pbx_weight *W, int64_t rows, int grad, size_t *bytes);
int pbx_linear_logprobs_dev(pbx_ctx *ctx, const pbx_weight *W, const float *dX, int64_t rows,
                            const int32_t *dTargets, float *dLogp, float *dEntropy, float *dLse,
                            void *work, size_t work_bytes);
/* The rows' gradient: dGradX[r] = dGradLogp[r] * d logp[r] / d x[r]
 *   = dGradLogp[r] * (W[dTargets[r]] - sum_v e^(logit_v - dLse[r]) W[v]),
 * 0 where a row's target is outside the vocabulary (padding), [rows][K], 16-byte aligned,
 * not dX itself.  dLse as pbx_linear_logprobs_dev gave it for these rows.  Logits are
 * computed again; of a target that is likelier than not, 1 - e^(logit - dLse) is taken as
 * the sum of the other entries' e^(logit_v - dLse), which keeps its bits however near to 1
 * the target comes.  Probabilities enter the second product with 22 bits, or with 2^-40 of
 * what the head's largest row would add where that is more, and weights with 22 bits
 * (2^-26 of the largest that the head's largest scale allows at least); sums are
 * held in f32 and come out the same in every call.  The weights stay as they are: they
 * have no gradient. */
int pbx_linear_logprobs_grad_dev(pbx_ctx *ctx, const pbx_weight *W, const float *dX, int64_t rows,
                                 const int32_t *dTargets, const float *dLse, const float *dGradLogp,
                                 float *dGradX, void *work, size_t work_bytes);

/* pbx_model_forward_batch that answers with log probabilities instead of n
 * rows of logits: row t's target is targets[t] (usually tokens[t + 1]; outside
 * the vocabulary: NaN).  Host arrays [n_tokens] or [n_tokens][top], as above;
 * any of the four outputs may be NULL (logp is needed with targets).  Waits for
 * its answers, so it is refused while the context's stream is captured, as
 * pbx_model_forward_kv is. */
int pbx_model_logprobs(pbx_model *m, const int32_t *tokens, int n_tokens, int start_pos,
                       const int32_t *targets, int top, float *logp, float *entropy,
                       int32_t *top_ids, float *top_logp);
/* One forward over the rows of a batch of sequences in a paged 8-bit cache (of
 * the model's context and with its layers, heads and head_dim; the model's own
 * cache is not touched): tokens[pbx_kv_batch_rows], packed as the batch's rows,
 * which must be the last of their sequences.  The cache's rotation counts:
 * PBX_ROPE_PAIRS with the model's rope_theta is the model's own.  Answers for
 * every row (all_rows), or for the last row of each sequence that has one, in
 * the batch's order: logits [rows][vocab], next_tokens (argmax), and the four
 * of pbx_model_logprobs with targets [rows]; each may be NULL.  At most
 * 65,535 rows.  Blocks until the answers are there.  A forward that fails leaves its rows of the cache undefined. */
int pbx_model_forward_kv(pbx_model *m, pbx_kv_batch *b, const int32_t *tokens, int all_rows,
                         float *logits, int32_t *next_tokens, const int32_t *targets, int top,
                         float *logp, float *entropy, int32_t *top_ids, float *top_logp);

#ifdef __cplusplus
}
#endif

#endif /* PBX_H */
